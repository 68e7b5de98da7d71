// Attention of the last T positions of every sequence over 8-bit pages.
//
//   o_r = sum_j p_rj sv_j V_j / sum_j p_rj,  p_rj = exp(scale sk_j (q_r . K_j) - max),
// K_j, V_j codes and sk_j, sv_j the scales of token j's page and kv head; row r
// stands at position ctx - T + t(r) and sees j up to it.
//
// HBM bounds it: every visible code is read once per kv head (D bytes per
// token each for K and V, half of a 16-bit cache), and all query rows of the
// head share it.  A warp streams units of 16 tokens through a private ring in
// shared memory by 16-byte asynchronous copies, several units ahead, and needs
// no barrier: lanes copy what they read themselves.
//
// The products run transposed, S^T = K Q^T and O^T = V^T P^T, as mma.sync
// m16n8k16: tokens (channels) are the 16 rows and 8 query rows the columns,
// so the 4 or 8 heads of a group fill a tile.  Contracted indexes may be
// permuted alike on both sides: a lane's 16 bytes of K serve four steps as
// they lie, and with tokens dealt to tile rows as token_of_row does, a lane's
// V bytes are A fragments after one byte permutation, and P^T is a B fragment
// after one 8 x 8 transposition.  Codes become fp16 exactly (e4m3 and int8
// both fit).  The query is scaled by a power of two per row and rounded to
// fp16 (exact for bf16 and fp16 down to 2^-29 of the row's largest channel,
// below that off by at most 2^-39 of it).
//
// P carries sv: w_rj = p_rj sv_j 2^(8 - M_r), with M_r a running maximum of
// log2(p sv) beside the softmax maximum m_r, so w fits fp16 whatever the
// scales are and is rounded relative to the largest contribution, not to the
// largest probability.  Both maxima move only when a value passes them by 2^7
// (exact: everything is divided by sums of the same terms), which leaves one
// vote per unit instead of shuffles and rescaling.
#include <cuda_fp16.h>

#include <climits>
#include <type_traits>

#include "attn_common.cuh"
#include "host_util.h"
#include "mma_sm80.cuh"
#include "sm100.cuh"

namespace attnb200 {
namespace attend8 {

constexpr int kWarps = 4;
constexpr int kRing = 65536;       // bytes of shared memory per CTA: kWarps rings
constexpr int kBatch = 32;         // units of a warp whose pages and scales its lanes hold
constexpr float kSlack = 7.f;      // a maximum moves when it is passed by this much (log2)
constexpr float kHead = 8.f;       // w <= 2^(kHead + kSlack) < 65504

struct Args {
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int32_t *table, *lens;
  const void* q;
  void* out;
  float *part_o, *part_lse;        // [seq][Hq * T][splits][D], [..][splits]
  int dtype, num_seqs, hq, hkv, t, num_blocks, bs, max_blocks, group, rows, row_groups, splits, chunk, max_context;
  float scale_log2;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t transposed8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Four codes -> fp16 pairs (0, 1) and (2, 3).
struct E4m3 {
  __device__ static void halves(uint32_t w, uint32_t* lo, uint32_t* hi) {
    asm("{.reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;}"
        : "=r"(*lo), "=r"(*hi)
        : "r"(w));
  }
  // 0xff in the place of each code that is NaN (0x7f or 0xff)
  __device__ static uint32_t nan_bytes(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }
};
struct Int8 {
  // 1024 + (c + 128) is fp16 0x6400 | (c ^ 0x80); minus 1152 it is c, exactly
  __device__ static void halves(uint32_t w, uint32_t* lo, uint32_t* hi) {
    const uint32_t x = w ^ 0x80808080u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 ha = __hsub2(*reinterpret_cast<const __half2*>(&a), bias);
    const __half2 hb = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
    *lo = *reinterpret_cast<const uint32_t*>(&ha);
    *hi = *reinterpret_cast<const uint32_t*>(&hb);
  }
  __device__ static uint32_t nan_bytes(uint32_t) { return 0; }
};

// Token (of 16) in row m of the K tile: rows 2a, 2a + 1 hold tokens 4a, 4a + 1
// and rows 8 + 2a, 9 + 2a tokens 4a + 2, 4a + 3, so that after the
// transposition lane (g, t) holds P of tokens 4t .. 4t + 3, whose V it loads.
__device__ __forceinline__ int token_of_row(int m) { return 4 * ((m & 7) >> 1) + (m & 1) + 2 * (m >> 3); }

__device__ __forceinline__ float load_q(const Args& a, long long at) {
  if (a.dtype == ATTN_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.q)[at]);
  if (a.dtype == ATTN_F16) return __half2float(reinterpret_cast<const __half*>(a.q)[at]);
  return reinterpret_cast<const float*>(a.q)[at];
}
__device__ __forceinline__ void store_out(void* out, int dtype, long long at, float x) {
  if (dtype == ATTN_BF16) reinterpret_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(x);
  else if (dtype == ATTN_F16) reinterpret_cast<__half*>(out)[at] = __float2half_rn(x);
  else reinterpret_cast<float*>(out)[at] = x;
}
__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// CTA = (kv head x group of 8 NT rows, split, sequence); its warps take the split's units in turn.
template <class F, int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT <= 2 ? 3 : 2) attend8_kernel(const __grid_constant__ Args a) {
  constexpr int KH = D / 64;                 // 64-byte halves of a row
  constexpr int MT = D / 16;                 // 16-channel tiles of O^T
  constexpr int kUnit = 32 * D;              // bytes of 16 tokens, K and V
  constexpr int S = kRing / kWarps / kUnit;  // ring stages
  constexpr int R = 8 * NT;
  const int split = blockIdx.y, seq = blockIdx.z;
  const int hk = blockIdx.x / a.row_groups, rg = blockIdx.x % a.row_groups;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  int ctx = max(a.lens[seq], 0);
  if (ctx > a.max_blocks * (long long)a.bs) {
    ctx = a.max_blocks * a.bs;  // (a sequence longer than its table row ends with the row)
    if (threadIdx.x == 0) atomicCAS(&g_notice, 0, kNoticeTableOverrun);
  }
  const int t0 = split * a.chunk;
  if (t0 >= ctx && split) return;
  const int t1 = (int)ll_min(ctx, (long long)t0 + a.chunk);
  const int units = (t1 - t0 + 15) / 16;

  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ float ml[kWarps][R][2];
  const uint32_t ring = smem_u32(smem) + warp * (kRing / kWarps);

  // Q^T as B fragments, a power of two per row (column g of tile n) taken out.  Four tiles of them are
  // 64 registers: they are read from shared memory instead, where all warps share them.
  constexpr bool QS = NT > 2;
  __shared__ uint2 qs[QS ? NT : 1][KH][4][QS ? 32 : 1];
  uint32_t qf[QS ? 1 : NT][KH][4][2];
  float cq[NT][2];   // rows 2t, 2t + 1 of each tile: softmax scale * log2 e / that power
  int last[NT][2];   // their last visible position + 1
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = rg * R + 8 * n + g;
    const bool there = row < a.rows;
    const int head = hk * a.group + (there ? row % a.group : 0), pos = there ? row / a.group : 0;
    const long long at = (((long long)seq * a.hq + head) * a.t + pos) * D;
    float x[KH][16], big = 0.f;
#pragma unroll
    for (int h = 0; h < KH; ++h)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        x[h][e] = there ? load_q(a, at + 64 * h + 16 * t + e) : 0.f;
        big = fmaxf(big, fabsf(x[h][e]));
      }
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    // the largest goes to [2^14, 2^15); infinite rows stay as they are
    int e2 = (int)(__float_as_uint(big) >> 23) - 127;
    e2 = big <= FLT_MAX ? max(e2, -100) - 14 : 0;
    const float mul = __uint_as_float((uint32_t)(127 - e2) << 23);
#pragma unroll
    for (int h = 0; h < KH; ++h)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t b0 = half_pair(x[h][4 * j] * mul, x[h][4 * j + 1] * mul);
        const uint32_t b1 = half_pair(x[h][4 * j + 2] * mul, x[h][4 * j + 3] * mul);
        if constexpr (QS) {
          if (warp == n % kWarps) qs[n][h][j][lane] = make_uint2(b0, b1);
        } else {
          qf[n][h][j][0] = b0;
          qf[n][h][j][1] = b1;
        }
      }
    const float c = a.scale_log2 * __uint_as_float((uint32_t)(127 + e2) << 23);
    const int lim = there ? ctx - a.t + pos + 1 : 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      cq[n][e] = __shfl_sync(0xffffffffu, c, 4 * (2 * t + e));
      last[n][e] = __shfl_sync(0xffffffffu, lim, 4 * (2 * t + e));
    }
  }

  if (QS) __syncthreads();

  float o[NT][MT][4];
  float m[NT][2], mo[NT][2], l[NT][2];  // the softmax maximum, that of p * sv, and this lane's part of the sum
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    m[n][0] = m[n][1] = mo[n][0] = mo[n][1] = -FLT_MAX;
    l[n][0] = l[n][1] = 0.f;
  }
  const int free_until = ctx - a.t + 1;  // tokens in front of this are visible to every row
  const long long row_bytes = (long long)a.hkv * D;

  for (int base = warp; base < units; base += kWarps * kBatch) {
    const int mine = min((units - base + kWarps - 1) / kWarps, kBatch);  // units base + kWarps * i of this warp
    long long first = 0;  // lane i: pool row of unit i's first token
    float lks = 0.f, lvs = 0.f;
    if (lane < mine) {
      const int tok = t0 + 16 * (base + kWarps * lane);
      const long long page = paged_phys_page(a.table[(long long)seq * a.max_blocks + tok / a.bs], a.num_blocks);
      first = page * a.bs + tok % a.bs;
      lks = a.ks[page * a.hkv + hk];
      lvs = a.vs[page * a.hkv + hk];
    }
    auto issue = [&](int i) {
      if (i < mine) {
        const long long r0 = __shfl_sync(0xffffffffu, first, i);
        const uint32_t dst = ring + (i % S) * kUnit + lane * 16;
        const uint8_t* kr = a.k + r0 * row_bytes + (long long)hk * D;
        const uint8_t* vr = a.v + r0 * row_bytes + (long long)hk * D;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int h = 0; h < KH; ++h)
            copy16(dst + (x * KH + h) * 512, kr + token_of_row(g + 8 * x) * row_bytes + 64 * h + 16 * t);
        if constexpr (D == 128) {
#pragma unroll
          for (int x = 0; x < 4; ++x) copy16(dst + (4 + x) * 512, vr + (4 * t + x) * row_bytes + 16 * g);
        } else {
          // rows of 64 bytes: piece (token, c) lies at c ^ (token / 4), free of bank conflicts for 8-byte reads
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int tok = 8 * x + (lane >> 2), c = lane & 3;
            copy16(ring + (i % S) * kUnit + 1024 + tok * 64 + ((c ^ (tok >> 2)) << 4), vr + tok * row_bytes + 16 * c);
          }
        }
      }
      copy_commit();
    };
#pragma unroll
    for (int i = 0; i < S - 1; ++i) issue(i);
    for (int i = 0; i < mine; ++i) {
      copy_wait<S - 2>();
      __syncwarp();
      issue(i + S - 1);
      const uint32_t slot = ring + (i % S) * kUnit;
      const int tok0 = t0 + 16 * (base + kWarps * i);
      const float ks = __shfl_sync(0xffffffffu, lks, i), vs = __shfl_sync(0xffffffffu, lvs, i);
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int h = 0; h < KH; ++h) {
        const uint4 ka = lds128(slot + lane * 16 + h * 512), kb = lds128(slot + lane * 16 + (KH + h) * 512);
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t f[4];
          F::halves(wa[j], &f[0], &f[2]);
          F::halves(wb[j], &f[1], &f[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if constexpr (QS) {
              const uint2 b = qs[n][h][j][lane];
              mma16816<false>(s[n], f, b.x, b.y);
            } else {
              mma16816<false>(s[n], f, qf[n][h][j][0], qf[n][h][j][1]);
            }
          }
        }
      }
      uint32_t vw[4][D / 32];  // tokens 4t + x: D / 8 bytes from channel g D / 8 on
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if constexpr (D == 128) {
          const uint4 w = lds128(slot + lane * 16 + (4 + x) * 512);
          vw[x][0] = w.x; vw[x][1] = w.y; vw[x][2] = w.z; vw[x][3] = w.w;
        } else {
          const uint2 w = lds64(slot + 1024 + (4 * t + x) * 64 + (((g >> 1) ^ t) << 4) + (g & 1) * 8);
          vw[x][0] = w.x; vw[x][1] = w.y;
        }
      }
      // scores in log2, and whether a maximum has to move
      const bool edge = tok0 + 16 > free_until;
      const float lv = fmaxf(lg2(fabsf(vs)), -100.f);
      bool seen[NT][4];
      bool move = false;
      const int ta = tok0 + token_of_row(g), tb = ta + 2;  // tokens of s[.][0, 1] and s[.][2, 3]
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = e & 1;
          s[n][e] *= ks * cq[n][r];
          seen[n][e] = !edge || (e < 2 ? ta : tb) < last[n][r];
          move = move || (seen[n][e] && (s[n][e] > m[n][r] + kSlack || s[n][e] + lv > mo[n][r] + kSlack));
        }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float mx = fmaxf(seen[n][r] ? s[n][r] : -FLT_MAX, seen[n][2 + r] ? s[n][2 + r] : -FLT_MAX);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float m_new = fmaxf(m[n][r], mx), mo_new = fmaxf(mo[n][r], mx + lv);
            const float fl = ex2(m[n][r] - m_new), fo = ex2(mo[n][r] - mo_new);
            m[n][r] = m_new;
            mo[n][r] = mo_new;
            l[n][r] *= fl;
#pragma unroll
            for (int i2 = 0; i2 < MT; ++i2) {
              o[n][i2][r] *= fo;
              o[n][i2][2 + r] *= fo;
            }
          }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = e & 1;
          const float p = seen[n][e] ? ex2(s[n][e] - m[n][r]) : 0.f;
          l[n][r] += p;
          s[n][e] = seen[n][e] ? p * (vs * ex2(m[n][r] - mo[n][r] + kHead)) : 0.f;  // w
        }
      if (edge) {
        // Slots behind the sequence may hold anything, NaN codes too: their V is zero.
        bool nan = false;
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int y = 0; y < D / 32; ++y) {
            if (tok0 + 4 * t + x >= ctx) vw[x][y] = 0;
            nan = nan || F::nan_bytes(vw[x][y]);
          }
        // A NaN among the values of the last T tokens must not meet the rows in front of it (0 * NaN): it is taken
        // out, and the rows that see it get it by hand.  (This lane's channels lie in its quad's V and in its own O.)
        if (a.t > 1 && __any_sync(0xffffffffu, nan)) {
#pragma unroll
          for (int y = 0; y < D / 32; ++y)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              int first = INT_MAX;
#pragma unroll
              for (int x = 3; x >= 0; --x)
                if (F::nan_bytes(vw[x][y]) & (0xffu << (8 * b))) first = tok0 + 4 * t + x;
              first = min(first, __shfl_xor_sync(0xffffffffu, first, 1));
              first = min(first, __shfl_xor_sync(0xffffffffu, first, 2));
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                  if (first < last[n][r]) o[n][2 * y + (b >> 1)][2 * (b & 1) + r] = NAN;
            }
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int y = 0; y < D / 32; ++y) vw[x][y] &= ~F::nan_bytes(vw[x][y]);
        }
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        pf[n][0] = transposed8x8(half_pair(s[n][0], s[n][1]));
        pf[n][1] = transposed8x8(half_pair(s[n][2], s[n][3]));
      }
#pragma unroll
      for (int y = 0; y < D / 32; ++y) {
        // (token 4t, token 4t + 1) pairs of channels 0, 1 | 2, 3 of the word, and the same of tokens 4t + 2, 4t + 3
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const uint32_t sel = z ? 0x7362u : 0x5140u;
          uint32_t f[4];
          F::halves(__byte_perm(vw[0][y], vw[1][y], sel), &f[0], &f[1]);
          F::halves(__byte_perm(vw[2][y], vw[3][y], sel), &f[2], &f[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<false>(o[n][2 * y + z], f, pf[n][0], pf[n][1]);
        }
      }
    }
    copy_wait<0>();
    __syncwarp();  // (the next batch starts on the ring again)
  }

  // ---- the warps' states into one ----
  __syncthreads();
  float* ow = reinterpret_cast<float*>(smem);  // [warp][R][D]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float sum = l[n][r];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      const float f = ex2(mo[n][r] - m[n][r] - kHead);
      const int row = 8 * n + 2 * t + r;
      float* at = ow + (warp * R + row) * D + g * (D / 8);
#pragma unroll
      for (int i = 0; i < MT; ++i)
        *reinterpret_cast<float2*>(at + 2 * i) = make_float2(o[n][i][r] * f, o[n][i][2 + r] * f);
      if (g == 0) {
        ml[warp][row][0] = m[n][r];
        ml[warp][row][1] = sum;
      }
    }
  __syncthreads();
  for (int row = warp; row < R; row += kWarps) {
    const int gr = rg * R + row;
    if (gr >= a.rows) break;
    float mx = -FLT_MAX;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, ml[w][row][0]);
    float tot = 0.f, acc[D / 32];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(ml[w][row][0] - mx);
      tot += f * ml[w][row][1];
#pragma unroll
      for (int e = 0; e < D / 32; ++e) acc[e] += f * ow[(w * R + row) * D + lane + 32 * e];
    }
    const float inv = tot == 0.f ? 0.f : 1.f / tot;  // (nothing visible: zeros)
    const long long orow = ((long long)seq * a.hq + hk * a.group + gr % a.group) * a.t + gr / a.group;
    if (a.splits == 1) {
#pragma unroll
      for (int e = 0; e < D / 32; ++e) store_out(a.out, a.dtype, orow * D + lane + 32 * e, acc[e] * inv);
    } else {
      const long long at = orow * a.splits + split;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) a.part_o[at * D + lane + 32 * e] = acc[e] * inv;
      if (lane == 0) a.part_lse[at] = tot == 0.f ? -INFINITY : mx + lg2(tot);
    }
  }
}

// Splits of one row: o = sum 2^(lse_i - M) o_i / sum 2^(lse_i - M).
template <int D>
__global__ void __launch_bounds__(D) join_kernel(const __grid_constant__ Args a) {
  pdl_wait_previous();
  const long long row = blockIdx.x;  // seq * Hq * T + head row
  const int seq = (int)(row / ((long long)a.hq * a.t)), d = threadIdx.x;
  const int ctx = (int)ll_min(max(a.lens[seq], 0), (long long)a.max_blocks * a.bs);
  const int need = (int)(((long long)ctx + a.chunk - 1) / a.chunk), n = min(need, a.splits);
  if (need > a.splits && d == 0) atomicCAS(&g_notice, 0, kNoticeContextOverrun);
  const float* lse = a.part_lse + row * a.splits;
  const float* po = a.part_o + row * a.splits * D + d;
  float mx = -FLT_MAX;
  for (int i = 0; i < n; ++i) mx = fmaxf(mx, lse[i]);
  float tot = 0.f, acc = 0.f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float f = ex2(lse[i] - mx);
    tot += f;
    acc += f * po[(long long)i * D];
  }
  store_out(a.out, a.dtype, row * D + d, tot == 0.f ? 0.f : acc / tot);
}

// -------------------------------------------------------------------- host --
static uintptr_t addr(const void* p) { return reinterpret_cast<uintptr_t>(p); }

static bool shape_ok(const attn_paged_attend8_params_t* p) {
  return p && (p->dtype == ATTN_F32 || p->dtype == ATTN_BF16 || p->dtype == ATTN_F16) &&
         (p->pool_format == ATTN_POOL_E4M3 || p->pool_format == ATTN_POOL_INT8) && p->num_seqs > 0 &&
         p->num_heads_kv > 0 && p->num_heads_q > 0 && p->num_heads_q % p->num_heads_kv == 0 && p->seq_q > 0 &&
         p->num_blocks > 0 && p->block_size > 0 && p->max_blocks_per_seq > 0 && p->head_dim > 0;
}

struct Plan {
  int nt, row_groups, splits, chunk;
};

static Plan make_plan(const attn_paged_attend8_params_t* p) {
  Plan pl;
  const long long rows = (long long)p->num_heads_q / p->num_heads_kv * p->seq_q;
  pl.nt = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
  pl.row_groups = (int)((rows + 8 * pl.nt - 1) / (8 * pl.nt));
  const long long ctx = ll_max(1, ll_min(p->max_context, (long long)p->max_blocks_per_seq * p->block_size));
  const long long ctas = (long long)p->num_seqs * p->num_heads_kv * pl.row_groups;
  const long long step = kWarps * 16, want = 148 * 3;
  long long chunk = step * kBatch;
  if (ctas * ((ctx + chunk - 1) / chunk) < want) chunk = ll_max(1, ctx * ctas / want / step) * step;
  // the partials stay within 1 GiB
  const long long row_bytes = (p->head_dim + 1) * 4ll * p->num_seqs * p->num_heads_q * p->seq_q;
  while (chunk < ctx && row_bytes * ((ctx + chunk - 1) / chunk) > (1ll << 30)) chunk *= 2;
  if (chunk >= ctx) chunk = (ctx + step - 1) / step * step;
  pl.chunk = (int)chunk;
  pl.splits = (int)((ctx + chunk - 1) / chunk);
  return pl;
}

}  // namespace attend8

bool attend8_take_status(int* status, int* notice) { return take_status_words(status, notice); }

}  // namespace attnb200

using namespace attnb200;

extern "C" {

size_t attn_paged_attend8_workspace_size(const attn_paged_attend8_params_t* p) {
  using namespace attend8;
  if (!shape_ok(p)) return 0;
  const Plan pl = make_plan(p);
  if (pl.splits == 1) return 0;
  const size_t rows = (size_t)p->num_seqs * p->num_heads_q * p->seq_q * pl.splits;
  return align256(rows * p->head_dim * 4) + align256(rows * 4);
}

int attn_paged_attend8(const attn_paged_attend8_params_t* p, void* stream) {
  using namespace attend8;
  if (!shape_ok(p) || !p->q || !p->out || !p->key_pool || !p->value_pool || !p->key_scales || !p->value_scales ||
      !p->block_table || !p->seq_lengths || p->max_context < 0)
    return ATTN_ERR_INVALID;
  if ((p->head_dim != 64 && p->head_dim != 128) || p->block_size % 16 ||
      (addr(p->key_pool) | addr(p->value_pool)) % 16)
    return ATTN_ERR_UNSUPPORTED;
  const Plan pl = make_plan(p);
  const long long rows = (long long)p->num_heads_q / p->num_heads_kv * p->seq_q;
  if (rows > INT_MAX / 2 || p->num_seqs > 65535 || pl.splits > 65535 ||
      (long long)p->num_heads_kv * pl.row_groups > INT_MAX ||
      (long long)p->num_seqs * p->num_heads_q * p->seq_q > INT_MAX)
    return ATTN_ERR_UNSUPPORTED;  // (grid dimensions)
  const size_t need = attn_paged_attend8_workspace_size(p);
  if (need && (!p->workspace || p->workspace_bytes < need)) return ATTN_ERR_WORKSPACE;
  if (need && addr(p->workspace) % 16) return ATTN_ERR_INVALID;
  Args a{};
  a.k = reinterpret_cast<const uint8_t*>(p->key_pool);
  a.v = reinterpret_cast<const uint8_t*>(p->value_pool);
  a.ks = p->key_scales; a.vs = p->value_scales;
  a.table = p->block_table; a.lens = p->seq_lengths;
  a.q = p->q; a.out = p->out; a.dtype = p->dtype;
  a.num_seqs = p->num_seqs; a.hq = p->num_heads_q; a.hkv = p->num_heads_kv; a.t = p->seq_q;
  a.num_blocks = p->num_blocks; a.bs = p->block_size; a.max_blocks = p->max_blocks_per_seq;
  a.group = p->num_heads_q / p->num_heads_kv; a.rows = (int)rows; a.row_groups = pl.row_groups;
  a.splits = pl.splits; a.chunk = pl.chunk; a.max_context = p->max_context;
  a.scale_log2 = p->softmax_scale * kLog2e;
  if (need) {
    const size_t n = (size_t)p->num_seqs * p->num_heads_q * p->seq_q * pl.splits;
    a.part_o = reinterpret_cast<float*>(p->workspace);
    a.part_lse = reinterpret_cast<float*>(reinterpret_cast<char*>(p->workspace) + align256(n * p->head_dim * 4));
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid(a.hkv * pl.row_groups, pl.splits, a.num_seqs);
#define RUN(F, D, NT)                                                                                     \
  do {                                                                                                    \
    auto* kern = &attend8_kernel<F, D, NT>;                                                               \
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing) != cudaSuccess)    \
      return ATTN_ERR_CUDA;                                                                               \
    kern<<<grid, kWarps * 32, kRing, st>>>(a);                                                            \
  } while (0)
#define BY_ROWS(F, D)            \
  do {                           \
    if (pl.nt == 1) RUN(F, D, 1); \
    else if (pl.nt == 2) RUN(F, D, 2); \
    else RUN(F, D, 4);           \
  } while (0)
  if (p->pool_format == ATTN_POOL_E4M3) {
    if (p->head_dim == 128) BY_ROWS(E4m3, 128);
    else BY_ROWS(E4m3, 64);
  } else {
    if (p->head_dim == 128) BY_ROWS(Int8, 128);
    else BY_ROWS(Int8, 64);
  }
#undef BY_ROWS
#undef RUN
  if (pl.splits == 1) return launch_status();
  const unsigned n = (unsigned)((long long)p->num_seqs * p->num_heads_q * p->seq_q);
  if (p->head_dim == 128) launch_overlapped(&join_kernel<128>, dim3(n), dim3(128), 0, st, a);
  else launch_overlapped(&join_kernel<64>, dim3(n), dim3(64), 0, st, a);
  return launch_status(2);
}

}  // extern "C"
