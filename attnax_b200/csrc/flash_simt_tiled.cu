// fp32 flash attention with sinks on register tiles (CUDA cores): forward,
// dQ, and dK/dV per query head.
//
// The one-row-per-thread-group kernels of flash_simt.cu read every K/V value
// from shared memory for a single multiply-add per row; they stay the path of
// everything that ran on them.  Here a block of 256 threads owns 64 x 64 (or 32
// x 64) score tiles, 4 x 4 per thread: 64 multiply-adds per 8 shared-memory
// vectors, so the FMA pipe bounds the products.  dK/dV of a kv head are computed
// per query head (a small batch then fills the GPU) and summed over the group
// in a fixed order.  Forward + backward, S1000 D128 W500, 4 sinks: B1 Hq8 Hkv1
// 7.5 -> 0.65 ms, B3 Hq32 Hkv8 18.2 -> 4.2 ms (about 30% of the FMA pipe; the
// rest is the masks' integer work and the unoverlapped tile loads).
#include <cfloat>

#include "attn_common.cuh"

namespace attnb200 {
namespace tiled {

constexpr int TB = 64;        // columns of a score tile
constexpr int kThreads = 256; // 16 x 16: thread (ty, tx) owns rows R ty.., columns tx + 16 j
constexpr int LP = TB + 4;    // row stride of a staged score tile

// R: rows per thread, 4 (row tiles of 64) or 2 (of 32, where 64-row tiles would leave SMs idle).
template <int D, int R>
struct Lay {
  static constexpr int TR = 16 * R;  // rows of a score tile
  static constexpr int LD = D + 4;   // row stride of a staged tile (16 rows apart in different banks)
  static constexpr int ROWS = TR * LD, COLS = TB * LD;
  static constexpr int NC = D / TB;  // float4 columns of an output row per thread
  static constexpr size_t fwd_smem = sizeof(float) * (ROWS + 2 * COLS + TR * LP);
  static constexpr size_t dq_smem = sizeof(float) * (2 * ROWS + 2 * COLS + TR * LP);
  static constexpr size_t dkv_smem = sizeof(float) * (2 * ROWS + 2 * COLS + 2 * TR * LP + 2 * TB);
  static_assert(dkv_smem <= 232448, "shared memory of a block");
};

struct Args {
  int B, Hq, Hkv, Sq, Skv, group;
  const float *q, *k, *v, *dout;
  float *out, *dq, *dk, *dv;
  long long qs[3], ks[3], vs[3], os[3], dos[3], dqs[3], dks[3], dvs[3];
  float* lse;                 // forward
  const float *lse2, *delta;  // backward, [B][Hq][Sq]
  float* part;                // [2][B][Hq][Skv][D]: dV and dK per query head
  float scale, sl2;
  attn_mask_t mask;
};

// Rows [r0, r0 + N) of a tensor into shared memory, zeros past its end.
template <int D, int N>
__device__ __forceinline__ void load_tile(float* dst, const float* src, long long stride, int r0, int rows) {
  for (int x = threadIdx.x; x < N * (D / 4); x += kThreads) {
    const int r = x / (D / 4), c = x % (D / 4) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r0 + r < rows) v = *reinterpret_cast<const float4*>(src + (r0 + r) * stride + c);
    *reinterpret_cast<float4*>(dst + r * (D + 4) + c) = v;
  }
}

// acc[i][j] = A[R ty + i] . B[tx + 16 j]
template <int D, int R>
__device__ __forceinline__ void rows_dot(const float* A, const float* B, int ty, int tx, float (&acc)[R][4]) {
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
#pragma unroll 4
  for (int d = 0; d < D; d += 4) {
    float4 a[R], b[4];
#pragma unroll
    for (int i = 0; i < R; ++i) a[i] = *reinterpret_cast<const float4*>(A + (R * ty + i) * (D + 4) + d);
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const float4*>(B + (tx + 16 * j) * (D + 4) + d);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[i][j] = fmaf(a[i].x, b[j].x, acc[i][j]);
        acc[i][j] = fmaf(a[i].y, b[j].y, acc[i][j]);
        acc[i][j] = fmaf(a[i].z, b[j].z, acc[i][j]);
        acc[i][j] = fmaf(a[i].w, b[j].w, acc[i][j]);
      }
  }
}

// acc[i][c] += sum_k P[R ty + i][k] * X[k][64 c + 4 tx ..]
template <int D, int R>
__device__ __forceinline__ void add_product(const float* P, const float* X, int ty, int tx,
                                            float4 (&acc)[R][D / TB]) {
#pragma unroll 2
  for (int k = 0; k < TB; k += 4) {
    float4 p[R];
#pragma unroll
    for (int i = 0; i < R; ++i) p[i] = *reinterpret_cast<const float4*>(P + (R * ty + i) * LP + k);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int c = 0; c < D / TB; ++c) {
        const float4 x = *reinterpret_cast<const float4*>(X + (k + e) * (D + 4) + c * TB + 4 * tx);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const float w = e == 0 ? p[i].x : e == 1 ? p[i].y : e == 2 ? p[i].z : p[i].w;
          acc[i][c].x = fmaf(w, x.x, acc[i][c].x);
          acc[i][c].y = fmaf(w, x.y, acc[i][c].y);
          acc[i][c].z = fmaf(w, x.z, acc[i][c].z);
          acc[i][c].w = fmaf(w, x.w, acc[i][c].w);
        }
      }
  }
}

template <int D, int R>
__device__ __forceinline__ void clear(float4 (&acc)[R][D / TB]) {
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int c = 0; c < D / TB; ++c) acc[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
}

template <int D, int R>
__device__ __forceinline__ void store_rows(float* dst, long long stride, int r0, int rows, int ty, int tx,
                                           const float4 (&acc)[R][D / TB], const float (&mul)[R]) {
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + R * ty + i;
    if (r >= rows) continue;
#pragma unroll
    for (int c = 0; c < D / TB; ++c)
      *reinterpret_cast<float4*>(dst + r * stride + c * TB + 4 * tx) =
          make_float4(acc[i][c].x * mul[i], acc[i][c].y * mul[i], acc[i][c].z * mul[i], acc[i][c].w * mul[i]);
  }
}

// Log2-domain score of (row, col), -FLT_MAX where dropped or outside.
__device__ __forceinline__ float score(const Args& a, float raw, float slope_l2, int b, int hq, int row, int col,
                                       bool partial) {
  if (row >= a.Sq || col >= a.Skv) return -FLT_MAX;
  return mask_score<true>(a.mask, raw, a.sl2, slope_l2, b, hq, row, col, a.Skv, partial);
}

template <int D, int R>
__global__ void __launch_bounds__(kThreads) fwd_kernel(const __grid_constant__ Args a) {
  using L = Lay<D, R>;
  extern __shared__ float sm[];
  float *sq = sm, *sk = sq + L::ROWS, *sv = sk + L::COLS, *sp = sv + L::COLS;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int q0 = (gridDim.x - 1 - blockIdx.x) * L::TR, hq = blockIdx.y, b = blockIdx.z, hkv = hq / a.group;
  const int q1 = min(q0 + L::TR, a.Sq);
  const float* K = a.k + b * a.ks[0] + hkv * a.ks[1];
  const float* V = a.v + b * a.vs[0] + hkv * a.vs[1];
  load_tile<D, L::TR>(sq, a.q + b * a.qs[0] + hq * a.qs[1], a.qs[2], q0, a.Sq);
  const float slope_l2 = a.mask.alibi_slopes ? a.mask.alibi_slopes[hq] * kLog2e : 0.f;
  float4 o[R][L::NC];
  clear<D, R>(o);
  float m[R], l[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    m[i] = -FLT_MAX;
    l[i] = 0.f;
  }
  int j_lo, j_hi;
  band_tile_range(a.mask, q0, q1, a.Skv, TB, &j_lo, &j_hi);
  const int n_sk = sink_tiles_before(sink_tile_count(a.mask, q1, a.Skv, TB), j_lo, j_hi);
  for (int t = j_lo - n_sk; t < j_hi; ++t) {
    const int j = t < j_lo ? t - (j_lo - n_sk) : t, k0 = j * TB;
    const int st = tile_state<true>(a.mask, nullptr, nullptr, 0, 0, b, q0, q1, k0, min(k0 + TB, a.Skv), TB);
    if (st == kSkip) continue;
    __syncthreads();
    load_tile<D, TB>(sk, K, a.ks[2], k0, a.Skv);
    load_tile<D, TB>(sv, V, a.vs[2], k0, a.Skv);
    __syncthreads();
    float s[R][4];
    rows_dot<D, R>(sq, sk, ty, tx, s);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float mx = m[i];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[i][c] = score(a, s[i][c], slope_l2, b, hq, q0 + R * ty + i, k0 + tx + 16 * c, st == kPartial);
        mx = fmaxf(mx, s[i][c]);
      }
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float alpha = exp2f(m[i] - mx);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float p = s[i][c] == -FLT_MAX ? 0.f : exp2f(s[i][c] - mx);
        sum += p;
        sp[(R * ty + i) * LP + tx + 16 * c] = p;
      }
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      l[i] = l[i] * alpha + sum;
      m[i] = mx;
#pragma unroll
      for (int c = 0; c < L::NC; ++c) {
        o[i][c].x *= alpha; o[i][c].y *= alpha; o[i][c].z *= alpha; o[i][c].w *= alpha;
      }
    }
    __syncwarp();  // (a row's 16 threads share a warp)
    add_product<D, R>(sp, sv, ty, tx, o);
  }
  float inv[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    inv[i] = l[i] == 0.f ? 0.f : 1.f / l[i];  // (0: no kept key; NaN scores make it NaN)
    const int r = q0 + R * ty + i;
    if (a.lse && tx == 0 && r < a.Sq)
      a.lse[((long long)b * a.Hq + hq) * a.Sq + r] = l[i] == 0.f ? -INFINITY : (m[i] + log2f(l[i])) * kLn2;
  }
  store_rows<D, R>(a.out + b * a.os[0] + hq * a.os[1], a.os[2], q0, a.Sq, ty, tx, o, inv);
}

template <int D, int R>
__global__ void __launch_bounds__(kThreads) dq_kernel(const __grid_constant__ Args a) {
  using L = Lay<D, R>;
  extern __shared__ float sm[];
  float *sq = sm, *sd = sq + L::ROWS, *sk = sd + L::ROWS, *sv = sk + L::COLS, *sp = sv + L::COLS;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int q0 = (gridDim.x - 1 - blockIdx.x) * L::TR, hq = blockIdx.y, b = blockIdx.z, hkv = hq / a.group;
  const int q1 = min(q0 + L::TR, a.Sq);
  const float* K = a.k + b * a.ks[0] + hkv * a.ks[1];
  const float* V = a.v + b * a.vs[0] + hkv * a.vs[1];
  load_tile<D, L::TR>(sq, a.q + b * a.qs[0] + hq * a.qs[1], a.qs[2], q0, a.Sq);
  load_tile<D, L::TR>(sd, a.dout + b * a.dos[0] + hq * a.dos[1], a.dos[2], q0, a.Sq);
  const float slope_l2 = a.mask.alibi_slopes ? a.mask.alibi_slopes[hq] * kLog2e : 0.f;
  float lse2[R], delta[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = q0 + R * ty + i;
    const long long at = ((long long)b * a.Hq + hq) * a.Sq + r;
    lse2[i] = r < a.Sq ? a.lse2[at] : INFINITY;
    delta[i] = r < a.Sq ? a.delta[at] : 0.f;
  }
  float4 dq[R][L::NC];
  clear<D, R>(dq);
  int j_lo, j_hi;
  band_tile_range(a.mask, q0, q1, a.Skv, TB, &j_lo, &j_hi);
  const int n_sk = sink_tiles_before(sink_tile_count(a.mask, q1, a.Skv, TB), j_lo, j_hi);
  for (int t = j_lo - n_sk; t < j_hi; ++t) {
    const int j = t < j_lo ? t - (j_lo - n_sk) : t, k0 = j * TB;
    const int st = tile_state<true>(a.mask, nullptr, nullptr, 0, 0, b, q0, q1, k0, min(k0 + TB, a.Skv), TB);
    if (st == kSkip) continue;
    __syncthreads();
    load_tile<D, TB>(sk, K, a.ks[2], k0, a.Skv);
    load_tile<D, TB>(sv, V, a.vs[2], k0, a.Skv);
    __syncthreads();
    float s[R][4], dp[R][4];
    rows_dot<D, R>(sq, sk, ty, tx, s);
    rows_dot<D, R>(sd, sv, ty, tx, dp);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float x = score(a, s[i][c], slope_l2, b, hq, q0 + R * ty + i, k0 + tx + 16 * c, st == kPartial);
        const float p = x == -FLT_MAX ? 0.f : exp2f(x - lse2[i]);
        sp[(R * ty + i) * LP + tx + 16 * c] = x == -FLT_MAX ? 0.f : p * (dp[i][c] - delta[i]);  // (dropped dP may be anything)
      }
    __syncwarp();
    add_product<D, R>(sp, sk, ty, tx, dq);
  }
  float mul[R];
#pragma unroll
  for (int i = 0; i < R; ++i) mul[i] = a.scale;
  store_rows<D, R>(a.dq + b * a.dqs[0] + hq * a.dqs[1], a.dqs[2], q0, a.Sq, ty, tx, dq, mul);
}

// dV and dK of 64 kv rows from one query head, into a.part.
template <int D, int R>
__global__ void __launch_bounds__(kThreads) dkv_kernel(const __grid_constant__ Args a) {
  using L = Lay<D, R>;
  extern __shared__ float sm[];
  float *sk = sm, *sv = sk + L::ROWS, *sq = sv + L::ROWS, *sd = sq + L::COLS, *sp = sd + L::COLS, *ss = sp + L::TR * LP;
  float *sl = ss + L::TR * LP, *se = sl + TB;  // lse2 and delta of the q tile
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int k0 = blockIdx.x * L::TR, hq = blockIdx.y, b = blockIdx.z, hkv = hq / a.group;
  const int k1 = min(k0 + L::TR, a.Skv);
  const float* Q = a.q + b * a.qs[0] + hq * a.qs[1];
  const float* G = a.dout + b * a.dos[0] + hq * a.dos[1];
  load_tile<D, L::TR>(sk, a.k + b * a.ks[0] + hkv * a.ks[1], a.ks[2], k0, a.Skv);
  load_tile<D, L::TR>(sv, a.v + b * a.vs[0] + hkv * a.vs[1], a.vs[2], k0, a.Skv);
  const float slope_l2 = a.mask.alibi_slopes ? a.mask.alibi_slopes[hq] * kLog2e : 0.f;
  float4 dk[R][L::NC], dv[R][L::NC];
  clear<D, R>(dk);
  clear<D, R>(dv);
  for (int q0 = 0; q0 < a.Sq; q0 += TB) {
    const int q1 = min(q0 + TB, a.Sq);
    const int st = tile_state<true>(a.mask, nullptr, nullptr, 0, 0, b, q0, q1, k0, k1, L::TR);
    if (st == kSkip) continue;
    __syncthreads();
    load_tile<D, TB>(sq, Q, a.qs[2], q0, a.Sq);
    load_tile<D, TB>(sd, G, a.dos[2], q0, a.Sq);
    if (threadIdx.x < TB) {
      const int r = q0 + threadIdx.x;
      const long long at = ((long long)b * a.Hq + hq) * a.Sq + r;
      sl[threadIdx.x] = r < a.Sq ? a.lse2[at] : INFINITY;
      se[threadIdx.x] = r < a.Sq ? a.delta[at] : 0.f;
    }
    __syncthreads();
    float s[R][4], dp[R][4];
    rows_dot<D, R>(sk, sq, ty, tx, s);   // S^T: rows are kv, columns q
    rows_dot<D, R>(sv, sd, ty, tx, dp);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int e = tx + 16 * c;
        const float x = score(a, s[i][c], slope_l2, b, hq, q0 + e, k0 + R * ty + i, st == kPartial);
        const float p = x == -FLT_MAX ? 0.f : exp2f(x - sl[e]);
        sp[(R * ty + i) * LP + e] = p;
        ss[(R * ty + i) * LP + e] = x == -FLT_MAX ? 0.f : p * (dp[i][c] - se[e]);
      }
    __syncwarp();
    add_product<D, R>(sp, sd, ty, tx, dv);
    add_product<D, R>(ss, sq, ty, tx, dk);
  }
  float one[R], mul[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    one[i] = 1.f;
    mul[i] = a.scale;
  }
  float* part = a.part + ((long long)b * a.Hq + hq) * a.Skv * D;
  store_rows<D, R>(part, D, k0, a.Skv, ty, tx, dv, one);
  store_rows<D, R>(part + (long long)a.B * a.Hq * a.Skv * D, D, k0, a.Skv, ty, tx, dk, mul);
}

// Sum over a kv head's query heads, in their order.
template <int D>
__global__ void __launch_bounds__(256) group_sum_kernel(const __grid_constant__ Args a) {
  const int r = blockIdx.x * (256 / (D / 4)) + threadIdx.x / (D / 4), c = threadIdx.x % (D / 4) * 4;
  const int hkv = blockIdx.y, b = blockIdx.z % a.B, which = blockIdx.z / a.B;  // dV, dK
  if (r >= a.Skv) return;
  const float* p = a.part + (long long)which * a.B * a.Hq * a.Skv * D +
                   ((long long)b * a.Hq + hkv * a.group) * a.Skv * D + (long long)r * D + c;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int g = 0; g < a.group; ++g) {
    const float4 x = *reinterpret_cast<const float4*>(p + (long long)g * a.Skv * D);
    s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
  }
  float* dst = which ? a.dk + b * a.dks[0] + hkv * a.dks[1] + r * a.dks[2] : a.dv + b * a.dvs[0] + hkv * a.dvs[1] + r * a.dvs[2];
  *reinterpret_cast<float4*>(dst + c) = s;
}

}  // namespace tiled
}  // namespace attnb200
