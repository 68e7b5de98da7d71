// Attention of the last T positions of every sequence over 8-bit pages.
//
//   o_r = sum_j p_rj sv_j V_j / sum_j p_rj,  p_rj = exp(scale sk_j (q_r . K_j) - max),
// K_j, V_j codes and sk_j, sv_j the scales of token j's page and kv head; row r
// stands at position ctx - T + t(r) and sees j up to it.
//
// HBM bounds it: every visible code is read once per kv head (D bytes per
// token each for K and V, half of a 16-bit cache), and all query rows of the
// head share it.  A warp streams units of 16 tokens by TMA through a private
// ring in shared memory, several units ahead, and shares no barrier with the
// other warps (64 sequences of 512 to 32768 tokens: 186 us, 5.5 TB/s; 16-byte
// copies by the lanes took 225).
//
// The products run transposed, S^T = K Q^T and O^T = V^T P^T, as mma.sync
// m16n8k16: tokens (channels) are the 16 rows and 8 query rows the columns,
// so the 4 or 8 heads of a group fill a tile.  Contracted indexes may be
// permuted alike on both sides: a lane's 16 bytes of K serve four steps as
// they lie, and with tokens dealt to tile rows as token_of_row does, a lane's
// V bytes are A fragments after one byte permutation, and P^T is a B fragment
// after one 8 x 8 transposition.  Codes become fp16 exactly (e4m3 and int8
// both fit).  The query is scaled by a power of two per row and rounded to
// fp16 (exact for bf16 and fp16 down to 2^-28 of the row's largest channel,
// below that off by at most 2^-39 of it; fp32 channels keep 11 bits, which is
// what P keeps too: a second product for their rest would leave P's rounding).
//
// P carries sv: w_rj = p_rj sv_j 2^(8 - M_r), with M_r a running maximum of
// log2(p sv) beside the softmax maximum m_r, so w fits fp16 whatever the
// scales are and is rounded relative to the largest contribution, not to the
// largest probability.  Both maxima move only when a value passes them by 2^7
// (exact: everything is divided by sums of the same terms), which leaves one
// vote per unit instead of shuffles and rescaling.  w is p times one factor
// sv 2^(8 + m - M); where that passes 2^(8 + kFar), w comes from an exponential
// of its own (the factor would pass fp32 in the end, and p its lower end).
// Such a p is below 2^(7 - kFar), which a sum of at least one does not hold.
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
constexpr int kSmem = kRing + 1024;  // (aligned by hand for the swizzle)
constexpr int kBatch = 32;         // units of a warp whose pages and scales its lanes hold
constexpr float kSlack = 7.f;      // a maximum moves when it is passed by this much (log2)
constexpr float kHead = 8.f;       // w <= 2^(kHead + kSlack) < 65504
constexpr float kFar = 64.f;       // log2(sv) + m - M from which w is formed without p

struct Args {
  const float *ks, *vs;
  const int32_t *table, *lens;
  const void* q;
  void* out;
  float *part_o, *part_lse;        // [seq][Hq * T][splits][D], [..][splits]
  int dtype, num_seqs, hq, hkv, t, num_blocks, bs, max_blocks, group, rows, row_groups, splits, chunk, max_context;
  float scale_log2;
};

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
// The page of sequence `seq`'s token `tok`.  An entry that is no page (freed by a window, or out
// of range) has nothing to read: `there` turns false, a notice is left, and the caller takes NaN for the scales, so that
// the rows which see such a token are NaN instead of another sequence's.
__device__ __forceinline__ long long page_of(const Args& a, int seq, int tok, bool* there) {
  const int e = a.table[(long long)seq * a.max_blocks + tok / a.bs];
  *there = e >= 0 && e < a.num_blocks;
  if (!*there) atomicCAS(&g_notice, 0, kNoticePageList);
  return *there ? e : 0;
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
  // 16 codes times 2^kShift as fp16, two 16-byte pieces: the bits of a code are those of an fp16 whose exponent is
  // biased by eight more, subnormal ones too.  Three integer steps a pair instead of a conversion on the unit that the
  // exponentials need.  NaN is put in where there is one.
  static constexpr float kShift = -8.f, kUnshift = 256.f;
  __device__ static void pairs(uint32_t w, uint32_t* lo, uint32_t* hi) {
    // (bytes with their signs spread above them, then seven up; what spills over and the second sign bit are masked)
    uint32_t a, b;
    asm("prmt.b32 %0, %1, 0, 0x9180;" : "=r"(a) : "r"(w));
    asm("prmt.b32 %0, %1, 0, 0xb3a2;" : "=r"(b) : "r"(w));
    *lo = (a << 7) & 0xbf80bf80u;
    *hi = (b << 7) & 0xbf80bf80u;
  }
  __device__ static void wide16(const uint4& w, uint4& lo, uint4& hi) {
    pairs(w.x, &lo.x, &lo.y);
    pairs(w.y, &lo.z, &lo.w);
    pairs(w.z, &hi.x, &hi.y);
    pairs(w.w, &hi.z, &hi.w);
    const uint32_t full = 0x7f7f7f7fu, one = 0x01010101u;
    if ((((w.x & full) + one) | ((w.y & full) + one) | ((w.z & full) + one) | ((w.w & full) + one)) & 0x80808080u) {
      const uint32_t n0 = nan_bytes(w.x), n1 = nan_bytes(w.y), n2 = nan_bytes(w.z), n3 = nan_bytes(w.w);
      nan_pair(n0, &lo.x, &lo.y);
      nan_pair(n1, &lo.z, &lo.w);
      nan_pair(n2, &hi.x, &hi.y);
      nan_pair(n3, &hi.z, &hi.w);
    }
  }
  // fp16 NaN where a code's byte of `bad` is set
  __device__ static void nan_pair(uint32_t bad, uint32_t* lo, uint32_t* hi) {
    *lo |= __byte_perm(bad, 0, 0x1100) & 0x7fff7fffu;
    *hi |= __byte_perm(bad, 0, 0x3322) & 0x7fff7fffu;
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
  static constexpr float kShift = 0.f, kUnshift = 1.f;
  __device__ static void wide16(const uint4& w, uint4& lo, uint4& hi) {
    halves(w.x, &lo.x, &lo.y);
    halves(w.y, &lo.z, &lo.w);
    halves(w.z, &hi.x, &hi.y);
    halves(w.w, &hi.z, &hi.w);
  }
  __device__ static uint32_t nan_bytes(uint32_t) { return 0; }
};

// The x-th of the four tokens (of a unit's 16) whose V lane (g, t) holds.  Rows 2a + e of the K tile hold token
// (a, e) and rows 8 + 2a + e token (a, 2 + e), so that after its transposition P meets them.  Which tokens these are
// is free; with these the 16-byte reads of K are free of bank conflicts on the swizzled tile.
template <int D>
__device__ __forceinline__ int token_of(int t, int x) {
  return D == 128 ? t + 4 * x : 2 * t + (x & 1) + 8 * (x >> 1);
}
// Byte of 16-byte piece c of a token in a unit's K or V tile (rows of 128 bytes, 128-byte swizzle; rows of 64, 64-byte).
template <int D>
__device__ __forceinline__ uint32_t place(int token, int c) {
  return D == 128 ? token * 128 + ((c ^ (token & 7)) << 4) : token * 64 + ((c ^ ((token >> 1) & 3)) << 4);
}

// 16 channels of the query as floats; rows start on 32 bytes.  (The loads are behind no branch: what it would move
// behind itself waits for them one by one.)
__device__ __forceinline__ void load_q16(const Args& a, long long at, float (&x)[16]) {
  const int elem = a.dtype == ATTN_F32 ? 4 : 2;
  const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.q) + at * elem);
  const uint4 w[4] = {p[0], p[1], p[elem == 4 ? 2 : 0], p[elem == 4 ? 3 : 1]};
  if (elem == 4) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      x[4 * c] = __uint_as_float(w[c].x);
      x[4 * c + 1] = __uint_as_float(w[c].y);
      x[4 * c + 2] = __uint_as_float(w[c].z);
      x[4 * c + 3] = __uint_as_float(w[c].w);
    }
    return;
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const uint32_t h[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (a.dtype == ATTN_BF16) {
        x[8 * c + 2 * e] = __uint_as_float(h[e] << 16);
        x[8 * c + 2 * e + 1] = __uint_as_float(h[e] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
        x[8 * c + 2 * e] = f.x;
        x[8 * c + 2 * e + 1] = f.y;
      }
    }
  }
}
// The power of two that is taken out of a row whose largest channel is `big`: that goes to [2^14, 2^15); rows with
// infinities stay as they are.
__device__ __forceinline__ int query_exponent(float big) {
  return big <= FLT_MAX ? max((int)(__float_as_uint(big) >> 23) - 127, -100) - 14 : 0;
}
// What turns products with such a row into scores in log2, but for the key scale.  With an infinity in it they are
// infinite or NaN for every key, and so the softmax is NaN; all of them -inf would pass for a row without keys.
__device__ __forceinline__ float query_factor(const Args& a, float big, int e2) {
  return big <= FLT_MAX ? a.scale_log2 * __uint_as_float((uint32_t)(127 + e2) << 23) : NAN;
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

// After a wait that ran out: what is in flight gets its time, with a limit, before its memory is given up.  (mbar_wait
// does not wait once a failure is recorded.)
__device__ __noinline__ void mbar_drain(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(bar, parity) && globaltimer() - t0 < ATTN_WAIT_NS) {
  }
}

}  // namespace attend8
}  // namespace attnb200

#include "attend8_tc.cuh"

namespace attnb200 {
namespace attend8 {

// CTA = (kv head x group of 8 NT rows, split, sequence); its warps take the split's units in turn.
template <class F, int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT <= 2 ? 3 : 2) attend8_kernel(
    const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Args a) {
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
  if (split == a.splits - 1 && t1 < ctx && threadIdx.x == 0) atomicCAS(&g_notice, 0, kNoticeContextOverrun);
  const int units = (t1 - t0 + 15) / 16;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ float ml[kWarps][R][2];
  const uint32_t ring = smem_u32(smem) + warp * (kRing / kWarps);
  __shared__ uint64_t bar[kWarps][S];
  const uint32_t bars = smem_u32(bar[warp]);
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < S; ++i) mbar_init(bars + 8 * i, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  __syncwarp();
  const int tk = token_of<D>(g >> 1, g & 1);  // the K tile's row g; row g + 8 is token tk + 8

  // The softmax maximum m and that of p sv, mo, of this lane's rows; up = 2^(kHead + m - mo); this lane's part of the sum.
  float o[NT][MT][4];
  float m[NT][2], mo[NT][2], up[NT][2], l[NT][2], apart = 0.f;  // apart: the largest m - mo, 0 at least
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    m[n][0] = m[n][1] = mo[n][0] = mo[n][1] = -FLT_MAX;
    up[n][0] = up[n][1] = 256.f;
    l[n][0] = l[n][1] = 0.f;
  }
  static_assert(kHead == 8.f, "up starts at 2^kHead, w of far pages has it as a factor");
  const int free_until = min(ctx - a.t + 1, t1);  // tokens of this split in front of it are visible to every row
  // This warp's units are warp + kWarps * j, j < mine.  Lane i holds the pool row and the scales of unit i of the
  // batch that is being loaded, and the scales of the batch that is being worked on.
  const int mine = max(units - warp + kWarps - 1, 0) / kWarps;
  int first = 0;
  float nks = 0.f, nvs = 0.f, lks = 0.f, lvs = 0.f;
  auto issue = [&](int j) {
    if (j >= mine) return;
    if (j % kBatch == 0 && j + lane < mine) {
      const int tok = t0 + 16 * (warp + kWarps * (j + lane));
      bool there;
      const long long page = page_of(a, seq, tok, &there);
      first = (int)(page * a.bs + tok % a.bs);
      nks = there ? a.ks[page * a.hkv + hk] : NAN;
      nvs = there ? a.vs[page * a.hkv + hk] : NAN;
    }
    const int row = __shfl_sync(0xffffffffu, first, j % kBatch);
    if (lane == 0) {
      const uint32_t dst = ring + (j % S) * kUnit, bar = bars + 8 * (j % S);
      mbar_expect_tx(bar, kUnit);
      tma_load_3d(dst, &tm_k, bar, 0, hk, row);
      tma_load_3d(dst + kUnit / 2, &tm_v, bar, 0, hk, row);
    }
  };
#pragma unroll
  for (int j = 0; j < S; ++j) issue(j);

  // Q^T as B fragments, a power of two per row (column g of tile n) taken out.  Those of several tiles
  // take too many registers: they are read from shared memory, where all warps share them.
  constexpr bool QS = NT > 1;
  __shared__ uint2 qs[QS ? NT : 1][KH][4][QS ? 32 : 1];
  uint32_t qf[QS ? 1 : NT][KH][4][2];
  const long long row0 = ((long long)seq * a.hq + hk * a.group) * a.t;  // the kv head's rows follow one another
  float cq[NT][2];   // rows 2t, 2t + 1 of each tile: softmax scale * log2 e / that power
  int last[NT][2];   // their last visible position of this split + 1
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = rg * R + 8 * n + g;
    const bool there = row < a.rows;
    const int pos = there ? row % a.t : 0;
    const long long at = (row0 + (there ? row : 0)) * D;
    float x[KH][16], big = 0.f;
#pragma unroll
    for (int h = 0; h < KH; ++h) {
      load_q16(a, at + 64 * h + 16 * t, x[h]);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        x[h][e] = there ? x[h][e] : 0.f;
        big = fmaxf(big, fabsf(x[h][e]));
      }
    }
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    const int e2 = query_exponent(big);
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
    const float c = query_factor(a, big, e2);
    const int lim = there ? min(ctx - a.t + pos + 1, t1) : 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      cq[n][e] = __shfl_sync(0xffffffffu, c, 4 * (2 * t + e));
      last[n][e] = __shfl_sync(0xffffffffu, lim, 4 * (2 * t + e));
    }
  }

  if (QS) __syncthreads();

  bool ok = true;
  int j = 0;
  for (; j < mine; ++j) {
    if (j % kBatch == 0) {
      lks = nks;
      lvs = nvs;
    }
    uint32_t vw[4][D / 32];  // V of this lane's four tokens: D / 8 bytes from channel g D / 8 on
    float s[NT][4];
    const uint32_t slot = ring + (j % S) * kUnit;
    const int tok0 = t0 + 16 * (warp + kWarps * j);
    const float ks = __shfl_sync(0xffffffffu, lks, j % kBatch), vs = __shfl_sync(0xffffffffu, lvs, j % kBatch);
    ok = ok && mbar_wait(bars + 8 * (j % S), (j / S) & 1, kStatusTimeoutLoad);
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int h = 0; h < KH; ++h) {
      const uint4 ka = lds128(slot + place<D>(tk, 4 * h + t)), kb = lds128(slot + place<D>(tk + 8, 4 * h + t));
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
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if constexpr (D == 128) {
        const uint4 w = lds128(slot + kUnit / 2 + place<D>(token_of<D>(t, x), g));
        vw[x][0] = w.x; vw[x][1] = w.y; vw[x][2] = w.z; vw[x][3] = w.w;
      } else {
        const uint2 w = lds64(slot + kUnit / 2 + place<D>(token_of<D>(t, x), g >> 1) + (g & 1) * 8);
        vw[x][0] = w.x; vw[x][1] = w.y;
      }
    }
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) break;
    __syncwarp();  // (all lanes have read the slots)
    issue(j + S);

    const bool edge = tok0 + 16 > free_until;
    // scores in log2; a maximum that one of them passes by kSlack moves
    bool move = false;
    const float lv = fmaxf(lg2(vs), -100.f);
    bool far = lv + apart > kFar;
    const int ta = tok0 + tk, tb = ta + 8;  // tokens of s[.][0, 1] and s[.][2, 3]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float c = ks * cq[n][r], top = m[n][r] + kSlack - fmaxf(0.f, lv + (m[n][r] - mo[n][r]));
#pragma unroll
        for (int e = r; e < 4; e += 2) {
          s[n][e] *= c;
          if (edge && (e < 2 ? ta : tb) >= last[n][r]) s[n][e] = -INFINITY;
          move = move || s[n][e] > top;
        }
      }
    if (__any_sync(0xffffffffu, move || far)) {
      far = __any_sync(0xffffffffu, far);
      apart = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float mx = fmaxf(fmaxf(s[n][r], s[n][2 + r]), -FLT_MAX);
#pragma unroll
          for (int w = 4; w <= 16; w *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
          const float m_new = fmaxf(m[n][r], mx), mo_new = fmaxf(mo[n][r], mx + lv);
          const float fl = ex2(m[n][r] - m_new), fo = ex2(mo[n][r] - mo_new);
          m[n][r] = m_new;
          mo[n][r] = mo_new;
          up[n][r] = ex2(m_new - mo_new + kHead);
          apart = fmaxf(apart, m_new - mo_new);
          l[n][r] *= fl;
#pragma unroll
          for (int i2 = 0; i2 < MT; ++i2) {
            o[n][i2][r] *= fo;
            o[n][i2][2 + r] *= fo;
          }
        }
    }
    auto weights = [&](auto far_rows) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float f = vs * up[n][r], from = m[n][r], in_sum = 1.f;
          if (decltype(far_rows)::value && lv + (m[n][r] - mo[n][r]) > kFar) {
            f = 256.f;
            from = mo[n][r] - lv;
            in_sum = 0.f;
          }
#pragma unroll
          for (int e = r; e < 4; e += 2) {
            const float p = ex2(s[n][e] - from);
            l[n][r] = decltype(far_rows)::value ? fmaf(p, in_sum, l[n][r]) : l[n][r] + p;
            s[n][e] = p * f;  // w
            if (edge && (e < 2 ? ta : tb) >= last[n][r]) s[n][e] = 0.f;  // (f may be NaN)
          }
        }
    };
    // (rare, and so asked for with the vote on the maxima, row by row only where some row may be so far; testing every
    // row of every unit cost 13 sequences of 5 tokens 27.3 us instead of 26.1)
    if (far) weights(std::true_type{});
    else weights(std::false_type{});
    if (edge) {
      // Slots behind the sequence may hold anything, NaN codes too: their V is zero.
      bool nan = false;
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < D / 32; ++y) {
          if (tok0 + token_of<D>(t, x) >= t1) vw[x][y] = 0;
          nan = nan || F::nan_bytes(vw[x][y]);
        }
      // A NaN among the values of the last T tokens must not meet the rows in front of it (0 * NaN): it is taken
      // out, and the rows that see it get it by hand.  (This lane's channels lie in its quad's V and in its own O.)
      if (a.t > 1 && __any_sync(0xffffffffu, nan)) {
#pragma unroll
        for (int y = 0; y < D / 32; ++y)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            int at = INT_MAX;
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (F::nan_bytes(vw[x][y]) & (0xffu << (8 * b))) at = min(at, tok0 + token_of<D>(t, x));
            at = min(at, __shfl_xor_sync(0xffffffffu, at, 1));
            at = min(at, __shfl_xor_sync(0xffffffffu, at, 2));
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int r = 0; r < 2; ++r)
                if (at < last[n][r]) o[n][2 * y + (b >> 1)][2 * (b & 1) + r] = NAN;
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
      // pairs (token 0, token 1) of channels 0, 1 | 2, 3 of the word, and the same of tokens 2, 3
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

  if (!ok)  // (a load that did not come: units j and on are in flight and get their time before the slots are given up)
    for (int u = j; u < min(j + S, mine); ++u) mbar_drain(bars + 8 * (u % S), (u / S) & 1);
  // ---- the warps' states into one ----
  if (!__syncthreads_and(ok)) return;
  float* ow = reinterpret_cast<float*>(smem);  // [warp][R][D]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float sum = l[n][r];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      // means, not sums: those of values near fp32's largest pass it
      const float f = sum == 0.f ? 0.f : __fdividef(ex2(mo[n][r] - m[n][r] - kHead), sum);
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
    for (int w = 0; w < kWarps; ++w) tot += ex2(ml[w][row][0] - mx) * ml[w][row][1];
    const float inv = tot == 0.f ? 0.f : 1.f / tot;  // (nothing visible: zeros)
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = 0.f;
    // A share is 2^(m_w - mx) sum_w / tot of the warp's mean.  That power meets the mean in two halves: alone it passes
    // the lower end of fp32 where the mean is large enough to count still.
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float half = ex2(0.5f * (ml[w][row][0] - mx)), c = half * ml[w][row][1] * inv;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) acc[e] = fmaf(ow[(w * R + row) * D + lane + 32 * e] * half, c, acc[e]);
    }
    const long long orow = row0 + gr;
    if (a.splits == 1) {
#pragma unroll
      for (int e = 0; e < D / 32; ++e) store_out(a.out, a.dtype, orow * D + lane + 32 * e, acc[e]);
    } else {
      const long long at = orow * a.splits + split;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) a.part_o[at * D + lane + 32 * e] = acc[e];
      if (lane == 0) a.part_lse[at] = tot == 0.f ? -INFINITY : mx + lg2(tot);
    }
  }
}

// Splits of a row: o = sum 2^(lse_i - M) o_i / sum 2^(lse_i - M), the terms times a power of two that keeps sums of the
// largest values in range, and in two halves as the warps' shares above (1 us of 115 for 8 sequences of 64 tokens; asking
// first whether a row needs them: 5).  `per_row` warps share a row's splits, each with a few in flight, and join through
// shared memory: one thread per channel that walks 40 splits took 9.3 us.
constexpr int kJoinWarps = 8;
template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const __grid_constant__ Args a, int per_row, int rows) {
  constexpr int E = D / 32;
  using V = typename std::conditional<E == 4, float4, float2>::type;
  __shared__ float acc_of[kJoinWarps][D + 1];
  pdl_wait_previous();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, part = warp % per_row;
  const int row = blockIdx.x * (kJoinWarps / per_row) + warp / per_row;  // seq * Hq * T + head row
  int n = 0;
  if (row < rows) {
    const int ctx = (int)ll_min(max(a.lens[row / (a.hq * a.t)], 0), (long long)a.max_blocks * a.bs);
    n = (int)ll_min(((long long)ctx + a.chunk - 1) / a.chunk, a.splits);
  }
  const float* lse = a.part_lse + (long long)row * a.splits;
  float mx = -FLT_MAX;
  for (int i = lane; i < n; i += 32) mx = fmaxf(mx, lse[i]);
#pragma unroll
  for (int w = 16; w; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
  float tot = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  const float least = __uint_as_float((uint32_t)(127 - 32 + __clz(n)) << 23);  // 2^-k with 2^k > n
  const V* po = reinterpret_cast<const V*>(a.part_o + (long long)row * a.splits * D) + lane;
#pragma unroll 4
  for (int i = part; i < n; i += per_row) {
    const float half = ex2(0.5f * (lse[i] - mx)), c = half * least;
    const V x = po[(long long)i * 32];
    tot = fmaf(half, c, tot);
    acc[0] = fmaf(x.x * half, c, acc[0]);
    acc[1] = fmaf(x.y * half, c, acc[1]);
    if constexpr (E == 4) {
      acc[2] = fmaf(x.z * half, c, acc[2]);
      acc[3] = fmaf(x.w * half, c, acc[3]);
    }
  }
  if (per_row > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) acc_of[warp][E * lane + e] = acc[e];
    if (lane == 0) acc_of[warp][D] = tot;
    __syncthreads();
    if (part) return;
    for (int w = 1; w < per_row; ++w) {
      tot += acc_of[warp + w][D];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += acc_of[warp + w][E * lane + e];
    }
  }
  if (row >= rows) return;
  const float inv = tot == 0.f ? 0.f : 1.f / tot;
#pragma unroll
  for (int e = 0; e < E; ++e) store_out(a.out, a.dtype, (long long)row * D + E * lane + e, acc[e] * inv);
}

// -------------------------------------------------------------------- host --
static uintptr_t addr(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// Map of an 8-bit pool [tokens, heads_kv, head_dim] with boxes of 16 tokens of one head, swizzled by their row length.
static bool make_map(CUtensorMap* m, const void* pool, long long tokens, int heads, int dim) {
  auto enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)tokens};
  cuuint64_t strides[2] = {(cuuint64_t)dim, (cuuint64_t)heads * dim};
  cuuint32_t box[3] = {(cuuint32_t)dim, 1, 16}, es[3] = {1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(pool), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static bool shape_ok(const attn_paged_attend8_params_t* p) {
  return p && (p->dtype == ATTN_F32 || p->dtype == ATTN_BF16 || p->dtype == ATTN_F16) &&
         (p->pool_format == ATTN_POOL_E4M3 || p->pool_format == ATTN_POOL_INT8) && p->num_seqs > 0 &&
         p->num_heads_kv > 0 && p->num_heads_q > 0 && p->num_heads_q % p->num_heads_kv == 0 && p->seq_q > 0 &&
         p->num_blocks > 0 && p->block_size > 0 && p->max_blocks_per_seq > 0 && p->head_dim > 0;
}

struct Plan {
  bool tc;
  int nt, row_groups, splits, chunk;
};

// From this many rows per kv head on the tcgen05 kernel runs: it converts the codes once for 256 rows, the other one
// for every 32.  Over the batches of make_plan's comment its time is 1.29 of the other one's at 32 rows, 0.99 at 48
// and 0.98 at 64; 8 sequences of 1000 to 16384 tokens, 8 kv heads: 128 rows 137 us against 86, 256 rows 229 against 119.
constexpr int kManyRows = 49;

static Plan make_plan(const attn_paged_attend8_params_t* p) {
  Plan pl;
  const long long rows = (long long)p->num_heads_q / p->num_heads_kv * p->seq_q;
  pl.tc = rows >= kManyRows;
  pl.nt = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
  const int group = pl.tc ? 256 : 8 * pl.nt;
  pl.row_groups = (int)((rows + group - 1) / group);
  const long long ctx = ll_max(1, ll_min(p->max_context, (long long)p->max_blocks_per_seq * p->block_size));
  const long long ctas = (long long)p->num_seqs * p->num_heads_kv * pl.row_groups;
  // tokens that splits come in, at most (but for what follows), CTAs that are wanted, steps of a split at least
  long long step, chunk, want, least;
  if (pl.tc) {
    // A CTA costs 14 us beside its tiles (3 to 3.7 us each) and writes 128 KB of partials: where one wave is not full,
    // splits of about what fills it, and longer ones (64 rows, 48 sequences: 368 -> 331 us) where there are many waves.
    // (The chunk is rounded down to tiles, so a few CTAs can be left to a second wave: one sequence of 16384 with 8 kv
    // heads and 256 rows has 176, and 72 us by these costs where splits of 1024 would have 44.)
    step = 128;
    least = 1;
    want = 148;
    chunk = ctas * ctx >= 148ll * 4 * 2048 ? 2048 : 1024;
  } else {
    // Lengths are ragged more often than not, so two waves if all were as long as the longest (of three CTAs an SM; with
    // 17 to 48 rows an SM holds two, and it is three); and at least 256 tokens
    // (four units a warp), for a shorter split costs more at its start and in the join than it brings.  Over 14 batches
    // (1 to 64 sequences of 100 to 100000 tokens, 2 to 8 kv heads), on average above the best choice of each batch at
    // 4, 8, 16 and 32 rows: 3, 5, 7 and 9%; four waves and 64 tokens 16, 19, 27 and 38%, one wave and 256 tokens 8, 10,
    // 13 and 8%, three waves 5, 6, 9 and 12%, two waves and 128 or 512 tokens 6 to 15% and 8 to 10%.
    step = kWarps * 16;
    least = 4;
    want = 148 * 3 * 2;
    chunk = step * kBatch;
  }
  if (ctas * ((ctx + chunk - 1) / chunk) < want) chunk = ll_max(least, ctx * ctas / want / step) * step;
  // the partials stay within 1 GiB
  const long long row_bytes = (p->head_dim + 1) * 4ll * p->num_seqs * p->num_heads_q * p->seq_q;
  while (chunk < ctx && row_bytes * ((ctx + chunk - 1) / chunk) > (1ll << 30)) chunk *= 2;
  if (chunk >= ctx) chunk = (ctx + step - 1) / step * step;
  pl.chunk = (int)ll_min(chunk, INT_MAX / step * step);
  pl.splits = (int)((ctx + pl.chunk - 1) / pl.chunk);
  return pl;
}

template <class F, int D>
static int launch_tc(const CUtensorMap& tk, const CUtensorMap& tv, const Args& a, dim3 grid, cudaStream_t st) {
  auto* kern = &attend8_tc_kernel<F, D>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Tc<D>::SMEM) != cudaSuccess)
    return ATTN_ERR_CUDA;
  kern<<<grid, Tc<D>::THREADS, Tc<D>::SMEM, st>>>(tk, tv, a);
  return ATTN_OK;
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
      (addr(p->key_pool) | addr(p->value_pool) | addr(p->q) | addr(p->out)) % 16)
    return ATTN_ERR_UNSUPPORTED;  // (TMA and vector accesses)
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
  const long long tokens = (long long)p->num_blocks * p->block_size;
  CUtensorMap tk, tv;
  if (tokens > INT_MAX) return ATTN_ERR_UNSUPPORTED;  // (coordinates are 32 bits)
  if (!make_map(&tk, p->key_pool, tokens, a.hkv, p->head_dim) || !make_map(&tv, p->value_pool, tokens, a.hkv, p->head_dim))
    return ATTN_ERR_CUDA;
  const dim3 grid(a.hkv * pl.row_groups, pl.splits, a.num_seqs);
#define RUN(F, D, NT)                                                                                     \
  do {                                                                                                    \
    auto* kern = &attend8_kernel<F, D, NT>;                                                               \
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)    \
      return ATTN_ERR_CUDA;                                                                               \
    kern<<<grid, kWarps * 32, kSmem, st>>>(tk, tv, a);                                                            \
  } while (0)
#define BY_ROWS(F, D)            \
  do {                           \
    if (pl.tc) {                 \
      const int rc = launch_tc<F, D>(tk, tv, a, grid, st); \
      if (rc != ATTN_OK) return rc; \
    } else if (pl.nt == 1) RUN(F, D, 1); \
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
  const int n = (int)((long long)p->num_seqs * p->num_heads_q * p->seq_q);
  const int per_row = pl.splits >= 16 ? 8 : pl.splits >= 8 ? 4 : pl.splits >= 4 ? 2 : 1;
  const dim3 blocks((n + kJoinWarps / per_row - 1) / (kJoinWarps / per_row));
  if (p->head_dim == 128) launch_overlapped(&join_kernel<128>, blocks, dim3(kJoinWarps * 32), 0, st, a, per_row, n);
  else launch_overlapped(&join_kernel<64>, blocks, dim3(kJoinWarps * 32), 0, st, a, per_row, n);
  return launch_status(2);
}

}  // extern "C"
