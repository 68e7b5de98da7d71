// Attention of several query rows per sequence over the paged KV cache:
//   * window: the rows are the last T positions of the cache and see a causal
//     sliding window plus the first tokens (sinks);
//   * tree: the rows are T drafted tokens, they see the whole context and the
//     drafted tokens on their own path (K/V of the drafts are not in the pages).
// No counterpart in the reference, which decodes with every row seeing the
// whole context (attnax/kernels/paged.py:17-84).
//
// Both are softmax(q k^T * scale | keep) v in one pass with a running maximum
// and sum, split over the visible tokens and joined by their log-sum-exp.  A
// row sum of exactly 0 means that the row saw nothing (zeros, lse -inf); a NaN
// score makes it NaN, and the row with it.  The
// rows of one kv head (its query heads x T) share every K/V read.  With up to
// 64 rows the work is bound by HBM (4 * rows flops per byte of K/V); wider
// trees approach the tensor cores' rate.
//   rows_mma_kernel  up to 32 rows: warp-level MMA on a TMA ring of 16- or
//                    32-token units, one or two row tiles of 16 per CTA
//   rows_tc_kernel   more rows: tcgen05 on 128-row x 128-token tiles gathered page by page by
//                    TMA, two CTAs per SM
//   rows_join_kernel joins the splits, its start hidden behind the end of the others; up to 8
//                    splits of rows_mma_kernel that all run at once form a cluster and join through
//                    each other's shared memory instead (one launch, no partials in memory; on
//                    tcgen05 a 64 KB tile per CTA makes that the slower way: 4 sequences of 8000, 64
//                    rows: 39.8 us joined by a launch, 46.3 us in clusters)
// Measured on one B200 (64 sequences of 512..32768 tokens, 8 kv heads of 128,
// bf16, GB/s of K/V): 4 rows 6556 / 5969 (warp MMA / tcgen05), 16 rows 6332 /
// 5787, 32 rows 5891 / 5692, 48 rows (four row tiles) 3295 / 5511; hence the
// border at 32.
#include <cfloat>

#include <atomic>

#include "attn_common.cuh"
#include "host_util.h"
#include "mma_sm80.cuh"
#include "sm100.cuh"

namespace attnb200 {
namespace rows {

constexpr int kMaxTree = 1024;   // drafted tokens per sequence
constexpr int kMmaRows = 32;     // rows of a kv head up to which rows_mma_kernel runs

struct Args {
  int N, Hq, Hkv, T, group, rows, row_groups;  // rows = group * T of one kv head
  int BS, max_blocks, num_blocks;
  long long window, sinks;
  int unit;                      // tokens of a TMA box
  int span_unit;                 // tokens of the units that splits count: `unit`, or the 128 of a tile
  int max_splits, split_units;   // units per split
  bool cluster;                  // the splits of a row are a cluster and join in it
  const void* q;
  const int32_t* block_table;
  const int32_t* seq_lens;
  const int32_t* parents;        // tree
  const int32_t* tree_lens;      // tree, or null
  float* part_o;    // [seq][Hkv * rows][max_splits][D], normalised
  float* part_lse;  // [seq][Hkv * rows][max_splits], log2 domain
  void* out;        // [seq][Hkv * rows][D]
  float sl2;
};

// What one sequence's rows see, in units of U tokens: units [0, n_sink) of the
// context, units [first, first + n_ctx) of the context, then n_draft units of
// drafted tokens.  Window: tokens in [lo, len) or below min(sinks, lo).
struct Span {
  int len, drafts, lo, first, n_sink, n_ctx, n_draft, total;
};

template <bool TREE>
__device__ __forceinline__ Span make_span(const Args& a, int seq, int U) {
  Span s;
  s.len = max(a.seq_lens[seq], 0);
  if (s.len > a.max_blocks * a.BS) {  // (no more tokens than the table row has pages for)
    atomicCAS(&g_notice, 0, kNoticeTableOverrun);
    s.len = a.max_blocks * a.BS;
  }
  s.drafts = 0;
  s.lo = 0;
  s.n_sink = 0;
  if (TREE) {
    s.drafts = a.tree_lens ? min(max(a.tree_lens[seq], 0), a.T) : a.T;
  } else {
    s.lo = (int)ll_max(0, (long long)s.len - a.T - a.window + 1);
  }
  s.first = s.lo / U;
  if (!TREE) s.n_sink = min((int)((ll_min(a.sinks, s.lo) + U - 1) / U), s.first);
  s.n_ctx = (s.len + U - 1) / U - s.first;
  s.n_draft = (s.drafts + U - 1) / U;
  s.total = s.n_sink + s.n_ctx + s.n_draft;
  return s;
}

// First token of unit v; `draft` says of which source.
__device__ __forceinline__ int unit_token(const Span& s, int v, int U, bool& draft) {
  draft = v >= s.n_sink + s.n_ctx;
  if (draft) return (v - s.n_sink - s.n_ctx) * U;
  return (v < s.n_sink ? v : s.first + v - s.n_sink) * U;
}

// Whether any row sees context token c.
template <bool TREE>
__device__ __forceinline__ bool ctx_visible(const Args& a, const Span& s, int c) {
  return c < s.len && (TREE || c >= s.lo || c < a.sinks);
}

__device__ __forceinline__ int page_of(const Args& a, int seq, int tok) {
  return (int)paged_phys_page(a.block_table[(long long)seq * a.max_blocks + tok / a.BS], a.num_blocks);
}

// Parent of drafted token t: negative, or in front of t.
__device__ __forceinline__ int parent_of(const int32_t* parents, int t) {
  const int p = parents[t];
  if (p >= t) {
    atomicCAS(&g_notice, 0, kNoticeTreeOrder);
    return -1;
  }
  return p;
}

// Splits this sequence really has (a length above max_context is cut to those planned).
__device__ __forceinline__ int split_count(const Args& a, const Span& s) {
  return min((s.total + a.split_units - 1) / a.split_units, a.max_splits);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Address of `p` (this CTA's shared memory) in CTA `rank` of the cluster.
template <typename T>
__device__ __forceinline__ T* in_cluster(T* p, int rank) {
  uint64_t out;
  asm("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
  return reinterpret_cast<T*>(out);
}

// One row joined from the splits' normalised rows `o` (this lane's D / 32
// values) and log-sum-exps `lse` in the CTAs [0, n) of the cluster, n <= 32.
template <int D, typename T, bool BF16>
__device__ __forceinline__ void join_in_cluster(float* o, float* lse, int n, int lane, T* out) {
  const float mine = lane < n ? *in_cluster(lse, lane) : -INFINITY;
  float mx = mine;
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
  const float w = mine == -INFINITY ? 0.f : ex2(mine - mx);  // (fmaxf skips NaN, this does not)
  float tot = 0.f, acc[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) acc[e] = 0.f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float* oi = in_cluster(o, i);
    const float wi = __shfl_sync(0xffffffffu, w, i);
    tot += wi;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = fmaf(wi, oi[e], acc[e]);
  }
  const float inv = tot == 0.f ? 0.f : 1.f / tot;
#pragma unroll
  for (int e = 0; e < D / 32; e += 2)
    *reinterpret_cast<uint32_t*>(out + e) = pack2(acc[e] * inv, acc[e + 1] * inv, BF16);
}

// ---------------------------------------------------- up to 32 query rows --
constexpr int NW = 4;  // consumer warps
constexpr int kMmaThreads = (NW + 1) * 32;

template <int D, int U>
struct MmaCfg {
  static constexpr int BOX = U * 128;            // U tokens x 64 features
  static constexpr int SLICE = (D / 64) * BOX;   // K or V of a unit
  static constexpr int STAGES = 65536 / (2 * SLICE);
  static constexpr int MS = D + 4;               // padded row of the merge buffer
  static constexpr int SMEM = 1024 + STAGES * 2 * SLICE + 2 * STAGES * 8;
  // After the ring has drained: the warps' states, then (cluster) up to 32 joined rows and their LSE.
  static constexpr int OFF_ROWS = NW * 16 * (MS + 2) * 4;
  static_assert(OFF_ROWS + kMmaRows * (D + 1) * 4 <= STAGES * 2 * SLICE, "the merge buffers fit the drained ring");
};

// RW row tiles of 16 per CTA, one per warp; the other NW / RW warps of a row
// tile take every (NW / RW)-th unit and are merged at the end.  64 KB of
// K/V in flight per CTA, three CTAs per SM.
template <bool BF16, int D, int U, int RW, bool TREE>
__global__ void __launch_bounds__(kMmaThreads, 3)
    rows_mma_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ CUtensorMap tm_dk, const __grid_constant__ CUtensorMap tm_dv,
                    const __grid_constant__ Args a) {
  using C = MmaCfg<D, U>;
  constexpr int S = C::STAGES, TW = NW / RW;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  const int hkv = blockIdx.x / a.row_groups, rg = blockIdx.x % a.row_groups;
  const int split = blockIdx.y, seq = blockIdx.z;
  const Span sp = make_span<TREE>(a, seq, U);
  const int n_split = split_count(a, sp);
  if (split >= n_split && split > 0 && !(a.cluster && n_split > 1)) return;
  if (split == 0 && threadIdx.x == 0 && sp.total > a.max_splits * a.split_units)
    atomicCAS(&g_notice, 0, kNoticeContextOverrun);
  const int v0 = split * a.split_units;
  const int n = max(0, min(sp.total - v0, a.split_units));

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t sb = (raw_base + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (sb - raw_base);
  float* rows_o = reinterpret_cast<float*>(smem + C::OFF_ROWS);  // [RW * 16][D], then their LSE
  float* rows_lse = rows_o + RW * 16 * D;
  const uint32_t k_base = sb, v_base = sb + S * C::SLICE, bar0 = sb + 2 * S * C::SLICE;
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (S + s); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row0 = ((long long)seq * a.Hkv + hkv) * a.rows;  // rows of q / out before this kv head's
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), RW);
    }
    fence_mbar_init();
  }
  __syncthreads();

  if (warp == NW) {
    if (lane == 0) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
    }
    // Pages of 32 units at a time are looked up by the 32 lanes.
    for (int i0 = 0; i0 < n; i0 += 32) {
      int row = 0;  // pool row (context) or token (draft) of this lane's unit
      bool draft = false;
      if (i0 + lane < n) {
        const int tok = unit_token(sp, v0 + i0 + lane, U, draft);
        row = draft ? tok : page_of(a, seq, tok) * a.BS + tok % a.BS;
      }
      bool ok = true;
      for (int j = 0; j < min(32, n - i0); ++j) {
        const int r = __shfl_sync(0xffffffffu, row, j), d = __shfl_sync(0xffffffffu, (int)draft, j);
        const int s = (i0 + j) % S;
        if (lane == 0 && ok) {
          ok = mbar_wait(empty(s), (((i0 + j) / S) & 1) ^ 1, kStatusTimeoutLoad);
          if (ok) {
            mbar_expect_tx(full(s), 2 * C::SLICE);
            for (int c = 0; c < D / 64; ++c) {
              const uint32_t kd = k_base + s * C::SLICE + c * C::BOX, vd = v_base + s * C::SLICE + c * C::BOX;
              if (TREE && d) {
                tma_load_4d(kd, &tm_dk, full(s), c * 64, r, hkv, seq);
                tma_load_4d(vd, &tm_dv, full(s), c * 64, r, hkv, seq);
              } else {
                tma_load_3d(kd, &tm_k, full(s), c * 64, hkv, r);
                tma_load_3d(vd, &tm_v, full(s), c * 64, hkv, r);
              }
            }
          }
        }
      }
      if (!__shfl_sync(0xffffffffu, (int)ok, 0)) break;
    }
  } else {
  pdl_launch_next();
  const int rt = warp % RW, tw = warp / RW;  // row tile, share of the units
  const int g = lane >> 2, tig = lane & 3;
  int pos[2];                          // window: position of the fragment rows; tree: drafted token
  bool row_ok[2];
  uint32_t anc[2] = {0, 0};            // tree: drafted tokens on the row's path (T <= rows <= 32)
  uint32_t qf[D / 16][4];              // A fragments: [k-step][row g lo, row g + 8 lo, row g hi, row g + 8 hi]
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = (rg * RW + rt) * 16 + g + 8 * h;
    const int t = r % a.T;
    row_ok[h] = r < a.rows && (!TREE || t < sp.drafts);
    pos[h] = TREE ? t : sp.len - a.T + t;
    const T* qr = reinterpret_cast<const T*>(a.q) + (row0 + r) * D;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      qf[kk][h] = row_ok[h] ? *reinterpret_cast<const uint32_t*>(qr + 16 * kk + 2 * tig) : 0u;
      qf[kk][2 + h] = row_ok[h] ? *reinterpret_cast<const uint32_t*>(qr + 16 * kk + 8 + 2 * tig) : 0u;
    }
  }
  if (TREE && v0 + n > sp.n_ctx) {
    // Lane x holds drafted token x: its path doubles in length with each step.
    int p = lane < sp.drafts ? parent_of(a.parents + (long long)seq * a.T, lane) : -1;  // (padding may hold anything)
    uint32_t path = 1u << lane;
#pragma unroll
    for (int x = 0; x < 5; ++x) {
      const uint32_t up = __shfl_sync(0xffffffffu, path, p & 31);
      const int pp = __shfl_sync(0xffffffffu, p, p & 31);
      if (p >= 0) path |= up;
      p = p >= 0 ? pp : -1;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t x = __shfl_sync(0xffffffffu, path, pos[h] & 31);
      anc[h] = row_ok[h] ? x : 0u;
    }
  }
  float o[D / 8][4];
#pragma unroll
  for (int x = 0; x < D / 8; ++x) o[x][0] = o[x][1] = o[x][2] = o[x][3] = 0.f;
  float m[2] = {-FLT_MAX, -FLT_MAX}, l[2] = {0.f, 0.f};
  const int mi = lane >> 3, ri = lane & 7;  // ldmatrix: matrix and row of this lane
  auto sw = [&](uint32_t base, int tok, int d) {  // swizzled [tok][d] of a unit's slice
    return base + (d >> 6) * C::BOX + tok * 128 + ((((d & 63) >> 3) ^ (tok & 7)) << 4);
  };
  bool ok = true;
  for (int i = tw; i < n; i += TW) {
    const int s = i % S;
    ok = __all_sync(0xffffffffu, mbar_wait(full(s), (i / S) & 1, kStatusTimeoutSoftmax));
    if (!ok) break;
    const uint32_t kst = k_base + s * C::SLICE, vst = v_base + s * C::SLICE;
    bool draft;
    const int tok0 = unit_token(sp, v0 + i, U, draft);
    // Kept whole by every row: no masks, every V row finite by contract.
    const bool whole = !draft && tok0 + U <= sp.len &&
                       (TREE || (tok0 + U - 1 <= sp.len - a.T && (tok0 >= sp.len - a.window || tok0 + U <= a.sinks)));
    bool zeroed = false;
#pragma unroll
    for (int g16 = 0; g16 < U; g16 += 16) {
      const int tok_a = tok0 + g16;
      if (!whole) {
        // V rows that nothing sees -> 0: P is 0 there, but a slot never written may hold NaN.
        // (Several row tiles write the same zeros.)
        for (int x = lane; x < 16 * (D / 8); x += 32) {
          const int r = x / (D / 8), u = x % (D / 8), tk = tok_a + r;
          if (draft ? tk >= sp.drafts : !ctx_visible<TREE>(a, sp, tk))
            *reinterpret_cast<uint4*>(smem + (sw(vst, g16 + r, u * 8) - sb)) = make_uint4(0, 0, 0, 0);
        }
        zeroed = true;
        __syncwarp();
      }
      float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t b[4];  // (tokens 0-7, d lo), (0-7, hi), (8-15, lo), (8-15, hi)
        ldsm_x4(b, sw(kst, g16 + 8 * (mi >> 1) + ri, 16 * kk + 8 * (mi & 1)));
        mma16816<BF16>(sc[0], qf[kk], b[0], b[1]);
        mma16816<BF16>(sc[1], qf[kk], b[2], b[3]);
      }
      // column (x, e) is token tok_a + 8x + 2*tig + (e & 1); e < 2: row g, else row g + 8
      if (!whole) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int tk = tok_a + 8 * x + 2 * tig + (e & 1), h = e >> 1;
            bool keep;
            if (TREE) keep = draft ? (tk < sp.drafts && ((anc[h] >> (tk & 31)) & 1)) : tk < sp.len;
            else keep = tk <= pos[h] && (pos[h] - tk < a.window || tk < a.sinks);
            if (!keep) sc[x][e] = -INFINITY;
          }
      }
      float alpha[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = fmaxf(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), fmaxf(sc[1][2 * h], sc[1][2 * h + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m[h], mx * a.sl2);
        alpha[h] = ex2(m[h] - m_new);
        m[h] = m_new;
      }
      float pr[2][4];
      float ps[2] = {0.f, 0.f};
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pr[x][e] = ex2(fmaf(sc[x][e], a.sl2, -m[e >> 1]));
          ps[e >> 1] += pr[x][e];
        }
      l[0] = l[0] * alpha[0] + ps[0];
      l[1] = l[1] * alpha[1] + ps[1];
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int x = 0; x < D / 8; ++x) {
          o[x][0] *= alpha[0]; o[x][1] *= alpha[0];
          o[x][2] *= alpha[1]; o[x][3] *= alpha[1];
        }
      }
      // P is rounded once to the cache's type, as the A operand of P V.
      const uint32_t pa[4] = {pack2(pr[0][0], pr[0][1], BF16), pack2(pr[0][2], pr[0][3], BF16),
                              pack2(pr[1][0], pr[1][1], BF16), pack2(pr[1][2], pr[1][3], BF16)};
#pragma unroll
      for (int np = 0; np < D / 16; ++np) {
        uint32_t b[4];  // (tokens 0-7, d tile 2np), (8-15, 2np), (0-7, 2np+1), (8-15, 2np+1)
        ldsm_x4_t(b, sw(vst, g16 + 8 * (mi & 1) + ri, 16 * np + 8 * (mi >> 1)));
        mma16816<BF16>(o[2 * np], pa, b[0], b[1]);
        mma16816<BF16>(o[2 * np + 1], pa, b[2], b[3]);
      }
    }
    if (zeroed) fence_proxy_async_smem();  // generic writes before the next TMA into this stage
    __syncwarp();
    if (lane == 0) mbar_arrive(empty(s));
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (!row_ok[h]) l[h] = 0.f;
  }
  // ---- merge the warps of a row tile through the drained ring ----
  named_bar_sync(1, NW * 32);
  constexpr int MS = C::MS;
  float* mo = reinterpret_cast<float*>(smem);  // [NW][16][MS]
  float* ml = mo + NW * 16 * MS;               // [NW][16][2]
#pragma unroll
  for (int x = 0; x < D / 8; ++x) {
    *reinterpret_cast<float2*>(mo + (warp * 16 + g) * MS + 8 * x + 2 * tig) = make_float2(o[x][0], o[x][1]);
    *reinterpret_cast<float2*>(mo + (warp * 16 + g + 8) * MS + 8 * x + 2 * tig) = make_float2(o[x][2], o[x][3]);
  }
  if (tig == 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      ml[(warp * 16 + g + 8 * h) * 2] = m[h];
      ml[(warp * 16 + g + 8 * h) * 2 + 1] = l[h];
    }
  }
  named_bar_sync(1, NW * 32);
  ok = __all_sync(0xffffffffu, ok);
  for (int j = warp; j < RW * 16; j += NW) {
    const int r = rg * RW * 16 + j;
    if (r >= a.rows || !ok) continue;
    const int t = j >> 4, jr = j & 15;  // row tile and row in it: warps t, t + RW, ...
    float mx = -FLT_MAX;
#pragma unroll
    for (int w = 0; w < TW; ++w) mx = fmaxf(mx, ml[((w * RW + t) * 16 + jr) * 2]);
    float lt = 0.f, acc[D / 32];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = 0.f;
#pragma unroll
    for (int w = 0; w < TW; ++w) {
      const int at = (w * RW + t) * 16 + jr;
      const float lw = ml[at * 2 + 1];
      const float f = lw == 0.f ? 0.f : ex2(ml[at * 2] - mx);  // (a row without keys holds o of nothing)
      lt += f * lw;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) acc[e] += f == 0.f ? 0.f : f * mo[at * MS + lane * (D / 32) + e];
    }
    const float inv = lt == 0.f ? 0.f : 1.f / lt;
    if (n_split <= 1) {
      T* orow = reinterpret_cast<T*>(a.out) + (row0 + r) * D + lane * (D / 32);
#pragma unroll
      for (int e = 0; e < D / 32; e += 2)
        *reinterpret_cast<uint32_t*>(orow + e) = pack2(acc[e] * inv, acc[e + 1] * inv, BF16);
    } else if (a.cluster) {
#pragma unroll
      for (int e = 0; e < D / 32; ++e) rows_o[j * D + lane * (D / 32) + e] = acc[e] * inv;
      if (lane == 0) rows_lse[j] = lt == 0.f ? -INFINITY : mx + lg2(lt);
    } else {
      const long long at = (row0 + r) * a.max_splits + split;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) a.part_o[at * D + lane * (D / 32) + e] = acc[e] * inv;
      if (lane == 0) a.part_lse[at] = lt == 0.f ? -INFINITY : mx + lg2(lt);
    }
  }
  }
  if (a.cluster && n_split > 1) {
    // Each CTA of the cluster joins a share of the rows; none leaves before its rows are read.
    __syncwarp();
    cluster_sync();
    if (warp < NW)
      for (int j = split + a.max_splits * warp; j < RW * 16; j += a.max_splits * NW) {
        const int r = rg * RW * 16 + j;
        if (r < a.rows)
          join_in_cluster<D, T, BF16>(rows_o + j * D + lane * (D / 32), rows_lse + j, n_split, lane,
                                      reinterpret_cast<T*>(a.out) + (row0 + r) * D + lane * (D / 32));
      }
    cluster_sync();
  }
}

// ----------------------------------------------- more than 32 query rows --
// CTA = NT tiles of 128 rows of one kv head x a split of its 128-token tiles.
// Warps 0-3 (and 4-7) run the softmax of a row tile (thread = row = TMEM lane),
// the next warp gathers the K/V tiles by TMA (one box per page piece, a lane
// each), the one behind it issues the MMAs; two more only complete the warpgroup
// that hands its registers to the softmax warps.  TMEM: S of tile x in [128 x,
// 128 x + 128), P over its first 64 columns, the O's behind the S's.
//   NT = 1 (up to 128 rows): a CTA's chain S -> softmax -> P V is serial; a second
//     CTA on the SM fills its gaps, which is enough to stay on HBM.
//   NT = 2 (more rows): the two tiles share every K/V tile and fill each other's
//     gaps (order P V_0, S_0, P V_1, S_1), one CTA per SM (2 sequences of 100000,
//     512 rows per kv head: 512 us with one tile per CTA, 488 us with two).
constexpr int BM = 128, BN = 128;
template <int D, int NT>
struct TcCfg {
  static constexpr int KCH = D / 64;
  static constexpr int STAGES = (NT == 1 ? 128 : 256) / D;  // 1 or 2 at D = 128, 2 or 4 at D = 64
  static constexpr int THREADS = 128 * (NT + 1);
  // Register split (setmaxnreg) of a CTA launched at REGS per thread.
  static constexpr int REGS = NT == 1 ? 128 : 168, PRODUCER_REGS = NT == 1 ? 56 : 104, SOFTMAX_REGS = 200;
  static_assert(128 * (PRODUCER_REGS + NT * SOFTMAX_REGS) == THREADS * REGS, "register split");
  static constexpr int Q_BYTES = KCH * BM * 128;  // one row tile
  static constexpr int KV_BYTES = KCH * BN * 128;
  static constexpr int OFF_K = NT * Q_BYTES;
  static constexpr int OFF_V = OFF_K + STAGES * KV_BYTES;
  static constexpr int OFF_BAR = OFF_V + STAGES * KV_BYTES;
  static constexpr int NBAR = 2 + 2 * NT + 4 * STAGES;
  static constexpr int OFF_TMEMPTR = OFF_BAR + NBAR * 8;
  static constexpr int OFF_PARENTS = OFF_TMEMPTR + 16;  // tree: the sequence's parents, 16 bits each
  static constexpr int SMEM = OFF_PARENTS + kMaxTree * 2 + 1024;
  static constexpr int CTAS = NT == 1 ? 2 : 1;  // per SM
  static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "resident CTAs");
  static constexpr uint32_t TMEM_COLS = 256 * NT;
  __host__ __device__ static constexpr uint32_t o_col(int x) { return 128 * NT + x * D; }
};

// The tile that position i of the split visits: context tiles in order, drafted
// tiles backwards, so that a row's walk up the tree goes on where it stopped.
__device__ __forceinline__ int tile_at(const Span& s, int v0, int n, int i) {
  const int ctx = s.n_sink + s.n_ctx, v = v0 + i;
  return v < ctx ? v : max(v0, ctx) + (v0 + n - 1 - v);
}

template <bool BF16, int D, int NT, bool TREE>
__global__ void __launch_bounds__(128 * (NT + 1), NT == 1 ? 2 : 1)
    rows_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_dk,
                   const __grid_constant__ CUtensorMap tm_dv, const __grid_constant__ Args a) {
  using C = TcCfg<D, NT>;
  constexpr int S = C::STAGES, kTma = 4 * NT, kMma = 4 * NT + 1;  // warps
  const int hkv = blockIdx.x / a.row_groups, rg = blockIdx.x % a.row_groups;
  const int split = blockIdx.y, seq = blockIdx.z;
  const Span sp = make_span<TREE>(a, seq, BN);
  const int n_split = split_count(a, sp);
  if (split >= n_split && split > 0) return;
  if (split == 0 && threadIdx.x == 0 && sp.total > a.max_splits * a.split_units)
    atomicCAS(&g_notice, 0, kNoticeContextOverrun);
  const int v0 = split * a.split_units;
  const int n = max(0, min(sp.total - v0, a.split_units));

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t sb = (raw_base + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (sb - raw_base);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bar0 = sb + C::OFF_BAR;
  const uint32_t q_full = bar0, o_done = bar0 + 8;
  auto s_full = [&](int x) { return bar0 + 8u * (2 + x); };
  auto p_full = [&](int x) { return bar0 + 8u * (2 + NT + x); };
  auto k_full = [&](int s) { return bar0 + 8u * (2 + 2 * NT + s); };
  auto v_full = [&](int s) { return bar0 + 8u * (2 + 2 * NT + S + s); };
  auto k_empty = [&](int s) { return bar0 + 8u * (2 + 2 * NT + 2 * S + s); };
  auto v_empty = [&](int s) { return bar0 + 8u * (2 + 2 * NT + 3 * S + s); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_TMEMPTR);
  int16_t* parents = reinterpret_cast<int16_t*>(smem + C::OFF_PARENTS);
  if (TREE && v0 + n > sp.n_ctx)  // this split holds drafted tokens (what the padding behind them holds is not read)
    for (int x = threadIdx.x; x < sp.drafts; x += C::THREADS)
      parents[x] = (int16_t)max(parent_of(a.parents + (long long)seq * a.T, x), -1);
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(o_done, 1);
    for (int x = 0; x < NT; ++x) {
      mbar_init(s_full(x), 1);
      mbar_init(p_full(x), 4);  // one arrival per softmax warp
    }
    for (int s = 0; s < S; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(v_full(s), 1);
      mbar_init(k_empty(s), 1);
      mbar_init(v_empty(s), 1);
    }
    fence_mbar_init();
  }
  if (warp == kMma) {
    tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;

  pdl_launch_next();
  if (warp >= kTma) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::PRODUCER_REGS));
    if (warp == kTma) {
      if (n > 0 && lane == 0) {
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
        mbar_expect_tx(q_full, NT * C::Q_BYTES);
        for (int x = 0; x < NT; ++x)
          for (int c = 0; c < C::KCH; ++c)
            tma_load_4d(sb + x * C::Q_BYTES + c * BM * 128, &tm_q, q_full, c * 64, (rg * NT + x) * BM, hkv, seq);
      }
      const int ub = a.unit;  // tokens per box: a page, or the power of two that divides it
      // Tile i: its first token, and this lane's box (pool row, or -1: nothing to load).
      auto boxes = [&](int i, int& tok0, bool& draft) {
        tok0 = unit_token(sp, tile_at(sp, v0, n, i), BN, draft);
        const int tok = tok0 + lane * ub;
        if (draft || lane * ub >= BN || tok >= sp.len || !(TREE || tok + ub > sp.lo || tok < a.sinks)) return -1;
        return page_of(a, seq, tok) * a.BS + tok % a.BS;
      };
      int tok0 = 0;
      bool draft = false;
      int row = n > 0 ? boxes(0, tok0, draft) : -1;
      for (int i = 0; i < n; ++i) {
        const int s = i % S;
        // (the next tile's pages are looked up while this one's stage is awaited: 8 sequences of 8000, 512
        // rows, 191 -> 182 us; bringing that tile into L2 as well was slower, 64 rows 776 -> 803 us)
        int next_tok0 = 0;
        bool next_draft = false;
        const int next_row = i + 1 < n ? boxes(i + 1, next_tok0, next_draft) : -1;
        const bool load = row >= 0;
        const uint32_t bytes = draft ? (uint32_t)C::KV_BYTES
                                     : __popc(__ballot_sync(0xffffffffu, load)) * (uint32_t)(ub * 128 * C::KCH);
        bool ok = true;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {  // K, then V
          const uint32_t bar = kv ? v_full(s) : k_full(s), free = kv ? v_empty(s) : k_empty(s);
          const uint32_t dst = sb + (kv ? C::OFF_V : C::OFF_K) + s * C::KV_BYTES;
          ok = ok && __all_sync(0xffffffffu, mbar_wait(free, ((i / S) & 1) ^ 1, kStatusTimeoutLoad));
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(bar, bytes);
          __syncwarp();
          if (TREE && draft) {
            if (lane == 0)
              for (int c = 0; c < C::KCH; ++c)
                tma_load_4d(dst + c * BN * 128, kv ? &tm_dv : &tm_dk, bar, c * 64, tok0, hkv, seq);
          } else if (load) {
            for (int c = 0; c < C::KCH; ++c)
              tma_load_3d(dst + c * BN * 128 + lane * ub * 128, kv ? &tm_v : &tm_k, bar, c * 64, hkv, row);
          }
        }
        if (!ok) break;
        row = next_row;
        tok0 = next_tok0;
        draft = next_draft;
      }
    } else if (warp == kMma && lane == 0 && n > 0) {
      constexpr int FMT = BF16 ? 1 : 0;
      constexpr uint32_t ID_S = idesc_f16(128, BN, FMT, 0, 0);
      constexpr uint32_t ID_O = idesc_f16(128, D, FMT, 0, 1);
      const uint64_t dQ = sdesc_sw128(sb, 16, 1024);
      const uint64_t dK = sdesc_sw128(sb + C::OFF_K, 16, 1024);
      const uint64_t dV = sdesc_sw128(sb + C::OFF_V, BN * 128, 1024);  // MN-major
      auto issue_s = [&](int x, int s) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_f16(tmem + x * 128, sdesc_add(dQ, x * C::Q_BYTES + (k >> 2) * BM * 128 + (k & 3) * 32),
                   sdesc_add(dK, s * C::KV_BYTES + (k >> 2) * BN * 128 + (k & 3) * 32), ID_S, k > 0 ? 1u : 0u);
        umma_commit(s_full(x));
      };
      auto issue_pv = [&](int x, int i) -> bool {
        if (!mbar_wait(p_full(x), i & 1, kStatusTimeoutMma)) return false;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)
          umma_f16_ts(tmem + C::o_col(x), tmem + x * 128 + k * 8, sdesc_add(dV, (i % S) * C::KV_BYTES + k * 16 * 128),
                      ID_O, (i > 0 || k > 0) ? 1u : 0u);
        return true;
      };
      // S of a row tile is issued behind its P V of the previous tile, which reads P from the same columns.
      bool ok = mbar_wait(q_full, 0, kStatusTimeoutMma);
      for (int i = 0; ok && i <= n; ++i) {
        if (i > 0) {
          ok = mbar_wait(v_full((i - 1) % S), ((i - 1) / S) & 1, kStatusTimeoutMma) && issue_pv(0, i - 1);
          if (!ok) break;
          if (NT == 1) umma_commit(v_empty((i - 1) % S));
        }
        if (i < n) {
          ok = mbar_wait(k_full(i % S), (i / S) & 1, kStatusTimeoutMma);
          if (!ok) break;
          tc_fence_after();
          issue_s(0, i % S);
        }
        if (NT == 2 && i > 0) {
          ok = issue_pv(1, i - 1);
          if (!ok) break;
          umma_commit(v_empty((i - 1) % S));
        }
        if (i < n) {
          if (NT == 2) issue_s(1, i % S);
          umma_commit(k_empty(i % S));
        }
      }
      if (ok) umma_commit(o_done);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFTMAX_REGS));
    const int x_tile = warp >> 2, rl = threadIdx.x & 127;  // row tile, row in it == TMEM lane
    const int r = (rg * NT + x_tile) * BM + rl;            // row of the kv head
    const int t = r % a.T;
    const bool row_ok = r < a.rows && (!TREE || t < sp.drafts);
    const int pos = sp.len - a.T + t;     // window: position of the row
    int walk = TREE && row_ok ? t : -1;   // tree: next token on the row's path
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_addr = lanes + x_tile * 128, o_addr = lanes + 128 * NT + x_tile * D;
    // A warp without rows (33 to 96 rows of a tile) leaves the exponentials to the others (64 rows:
    // the two idle warps' share of the SM was half of all).
    const bool idle = r - lane >= a.rows;
    // V rows that nothing sees -> 0: P is 0 there, but a slot never written (or a box never
    // loaded) may hold NaN.  Thread = token; with two row tiles both write the same zeros.
    auto clear_v = [&](int st, int i, int tok0, bool draft) -> bool {
      if (!__all_sync(0xffffffffu, mbar_wait(v_full(st), (i / S) & 1, kStatusTimeoutSoftmax))) return false;
      const int tk = tok0 + rl;
      if (draft ? tk >= sp.drafts : !ctx_visible<TREE>(a, sp, tk)) {
#pragma unroll
        for (int c = 0; c < C::KCH; ++c)
#pragma unroll
          for (int u = 0; u < 8; ++u)
            *reinterpret_cast<uint4*>(smem + C::OFF_V + st * C::KV_BYTES + c * BN * 128 + rl * 128 + u * 16) =
                make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async_smem();
      return true;
    };
    float m = -FLT_MAX, l = 0.f;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int st = i % S;
      bool draft;
      const int tok0 = unit_token(sp, tile_at(sp, v0, n, i), BN, draft);
      const bool whole =
          !draft && tok0 + BN <= sp.len &&
          (TREE || (tok0 + BN - 1 <= sp.len - a.T && (tok0 >= sp.len - a.window || tok0 + BN <= a.sinks)));
      uint32_t keep[4] = {0u, 0u, 0u, 0u};
      if (!whole) {
        if (TREE && draft) {
          while (walk >= tok0) {  // (tokens behind this tile were passed in the tiles behind it)
            const int x = walk - tok0;
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if ((x >> 5) == c) keep[c] |= 1u << (x & 31);
            walk = parents[walk];
          }
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const long long c0 = tok0 + c * 32;
            if (TREE) keep[c] = bit_range(0, sp.len - 1 - c0);
            else keep[c] = (bit_range(pos - a.window + 1 - c0, 31) | bit_range(0, a.sinks - 1 - c0)) & bit_range(0, pos - c0);
          }
        }
      }
      ok = __all_sync(0xffffffffu, mbar_wait(s_full(x_tile), i & 1, kStatusTimeoutSoftmax));
      if (!ok) break;
      tc_fence_after();
      if (idle) {
        // No rows here: P and O of these lanes may hold anything, the tile's V rows are still cleared below.
        if (!whole && !clear_v(st, i, tok0, draft)) { ok = false; break; }
        tc_fence_before();
        mbar_arrive_warp(p_full(x_tile));
        continue;
      }
      float x[BN];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&x[c * 32]));
      tmem_wait_ld();
      if (!whole) {
#pragma unroll
        for (int c = 0; c < BN; ++c)
          if (!((keep[c >> 5] >> (c & 31)) & 1u)) x[c] = -INFINITY;
        ok = clear_v(st, i, tok0, draft);
        if (!ok) break;
      }
      float mxp[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < BN; ++c) mxp[c & 3] = fmaxf(mxp[c & 3], x[c]);
      const float mx = fmaxf(fmaxf(mxp[0], mxp[1]), fmaxf(mxp[2], mxp[3])) * a.sl2;
      // The running maximum follows only jumps of more than 2^8 (P stays <= 256, exact after the final 1/l).
      float alpha = 1.f;
      if (mx > m + 8.f) {
        alpha = ex2(m - mx);
        m = mx;
      }
      const unsigned long long sc2 = f2_pack(a.sl2, a.sl2), nm2 = f2_pack(-m, -m);
      unsigned long long sum2[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          float x0, x1;
          f2_unpack(f2_fma(f2_pack(x[h * 64 + c], x[h * 64 + c + 1]), sc2, nm2), x0, x1);
          const float p0 = ex2(x0), p1 = ex2(x1);
          sum2[(c >> 1) & 1] = f2_add(sum2[(c >> 1) & 1], f2_pack(p0, p1));
          pk[c >> 1] = pack2(p0, p1, BF16);  // P rounded once to the cache's type
        }
        tmem_st32(s_addr + h * 32, pk);
      }
      float s0, s1, s2, s3;
      f2_unpack(sum2[0], s0, s1);
      f2_unpack(sum2[1], s2, s3);
      l = l * alpha + ((s0 + s1) + (s2 + s3));
      // P V of the previous tile is complete: S of this one was issued behind it.
      if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st32(o_addr + c * 32, o);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive_warp(p_full(x_tile));
    }
    if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait(o_done, 0, kStatusTimeoutSoftmax));
    if (ok) {
      tc_fence_after();
      if (!row_ok) l = 0.f;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const long long row = ((long long)seq * a.Hkv + hkv) * a.rows + r;
      const long long at = row * a.max_splits + split;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld32(o_addr + c * 32, o);
          tmem_wait_ld();
        }
        // (a row without keys may hold o of nothing: select, do not multiply)
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = l == 0.f ? 0u : __float_as_uint(__uint_as_float(o[e]) * inv);
        if (r >= a.rows) continue;
        if (n_split <= 1) {
          T* orow = reinterpret_cast<T*>(a.out) + row * D + c * 32;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            uint4 w;
            w.x = pack2(__uint_as_float(o[v * 8 + 0]), __uint_as_float(o[v * 8 + 1]), BF16);
            w.y = pack2(__uint_as_float(o[v * 8 + 2]), __uint_as_float(o[v * 8 + 3]), BF16);
            w.z = pack2(__uint_as_float(o[v * 8 + 4]), __uint_as_float(o[v * 8 + 5]), BF16);
            w.w = pack2(__uint_as_float(o[v * 8 + 6]), __uint_as_float(o[v * 8 + 7]), BF16);
            *reinterpret_cast<uint4*>(orow + v * 8) = w;
          }
        } else {
          float* po = a.part_o + at * D + c * 32;
#pragma unroll
          for (int v = 0; v < 8; ++v)
            *reinterpret_cast<uint4*>(po + v * 4) = make_uint4(o[v * 4], o[v * 4 + 1], o[v * 4 + 2], o[v * 4 + 3]);
        }
      }
      if (r < a.rows && n_split > 1) a.part_lse[at] = l == 0.f ? -INFINITY : m + lg2(l);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// Joins the splits of a row: o = sum 2^(lse_i - M) o_i / sum 2^(lse_i - M).  One warp per row;
// sequences with one split were written by their only CTA.
template <typename T, int D, bool TREE>
__global__ void __launch_bounds__(256) rows_join_kernel(const __grid_constant__ Args a) {
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), seq = blockIdx.y, lane = threadIdx.x & 31;
  if (row >= a.Hkv * a.rows) return;
  const Span sp = make_span<TREE>(a, seq, a.span_unit);  // (lengths: not written by the kernel in front)
  const int n = split_count(a, sp);
  pdl_wait_previous();  // (also where there is nothing to join: this kernel must not end before that one)
  if (n <= 1) return;
  const long long prow = (long long)seq * a.Hkv * a.rows + row;
  const float* lse = a.part_lse + prow * a.max_splits;
  const float* po = a.part_o + prow * a.max_splits * D + lane * (D / 32);
  float mx = -INFINITY;
  bool nan = false;  // (fmaxf skips NaN)
  for (int i = lane; i < n; i += 32) {
    mx = fmaxf(mx, lse[i]);
    nan = nan || lse[i] != lse[i];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  nan = __any_sync(0xffffffffu, nan);
  float tot = 0.f, acc[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) acc[e] = 0.f;
  if (mx != -INFINITY) {
    constexpr int B = 8;  // partials in flight
    for (int i0 = 0; i0 < n; i0 += 32) {
      const float wl = i0 + lane < n ? ex2(lse[i0 + lane] - mx) : 0.f;
      for (int j0 = 0; j0 < min(32, n - i0); j0 += B) {
        float x[B][D / 32];
#pragma unroll
        for (int j = 0; j < B; ++j)
#pragma unroll
          for (int e = 0; e < D / 32; ++e)
            x[j][e] = i0 + j0 + j < n ? po[(long long)(i0 + j0 + j) * D + e] : 0.f;
#pragma unroll
        for (int j = 0; j < B; ++j) {
          const float w = __shfl_sync(0xffffffffu, wl, j0 + j);
          tot += w;
#pragma unroll
          for (int e = 0; e < D / 32; ++e) acc[e] = fmaf(w, x[j][e], acc[e]);
        }
      }
    }
  }
  const float inv = nan ? NAN : tot > 0.f ? 1.f / tot : 0.f;
  T* orow = reinterpret_cast<T*>(a.out) + prow * D + lane * (D / 32);
#pragma unroll
  for (int e = 0; e < D / 32; e += 2)
    *reinterpret_cast<uint32_t*>(orow + e) =
        pack2(acc[e] * inv, acc[e + 1] * inv, std::is_same<T, __nv_bfloat16>::value);
}

// -------------------------------------------------------------------- host --
struct Plan {
  bool tc, cluster;
  int unit, span_unit, row_tiles, row_groups, max_splits, split_units;
  size_t part_lse, total;
};

// Tokens that a sequence's rows can see, at most.
static long long max_tokens(const attn_paged_params_t* p, bool tree, int64_t window, int64_t sinks) {
  const long long ctx = p->max_context;
  if (tree) return ctx;
  const long long w = window < ctx ? window + p->seq_q - 1 : ctx, s = sinks < ctx ? sinks : ctx;
  return ll_min(ctx, w + s);
}

// Splits: the number that ends first if every sequence is as long as it may be,
// counting waves of resident CTAs.  None under 128 tokens (one sequence of 2500 tokens, one
// row: 14.7 us at 128 or 256 tokens, 18.8 at 512, 31.0 at 1024), and none longer
// than keeps ragged batches even: 2048 tokens with few rows, where a partial is
// small next to its K/V; 4096 on tcgen05, whose partials are up to 128 rows x
// 512 bytes (96 rows: 5094 GB/s at 2048, 5381 at 4096; 256 rows: 1736 us and
// 1430 us).
// Splits that join in a cluster: as many as a cluster holds everywhere, and
// only where every CTA runs at once (a CTA of a short sequence waits for its
// cluster, which would keep the next wave's CTAs out).
static bool cluster_fits(bool tc, long long splits, long long waves) { return !tc && splits <= 8 && waves <= 1; }
// A CTA's start and its partial, and a launch of rows_join_kernel, in the time
// of so many tokens of a CTA (one sequence of 2500 tokens, one row: 10.2 us in
// 20 splits and a join, 12.5 us in a cluster of 8; of 1028 tokens: 9.0 and 8.4).
constexpr int kStartTokens = 256, kJoinTokens = 96;
// Many long sequences with many rows each have CTAs enough: there the longest
// split grows instead of the partials (8 sequences of 131072, 1024 drafts, 64
// heads: 39.5 ms and 9.3 GiB in splits of 4096, 33.1 ms and 0.8 GiB so).
constexpr long long kMaxPartials = 1ll << 30;

static Plan make_plan(const attn_paged_params_t* p, bool tree, int64_t window, int64_t sinks) {
  Plan w;
  const int rows = p->num_heads_q / p->num_heads_kv * p->seq_q;
  w.tc = rows > kMmaRows;
  if (w.tc) {
    w.unit = 128;
    while (p->block_size % w.unit != 0) w.unit /= 2;
    w.span_unit = BN;
    w.row_tiles = (rows > BM ? 2 : 1) * (BM / 16);
  } else {
    w.unit = w.span_unit = p->block_size % 32 == 0 ? 32 : 16;
    w.row_tiles = rows <= 16 ? 1 : 2;
  }
  w.row_groups = (rows + w.row_tiles * 16 - 1) / (w.row_tiles * 16);
  const long long tokens = max_tokens(p, tree, window, sinks), u = w.span_unit;
  // (window: the first and last unit of both pieces may be cut)
  const long long units = (tokens + u - 1) / u + (tree ? (p->seq_q + u - 1) / u : 3);
  const long long ctas = (long long)p->num_seqs * p->num_heads_kv * w.row_groups;
  const long long slots = (w.tc ? (rows > BM ? 1 : 2) : 3) * 148;
  const long long least = ll_max(128 / u, 1), most = (w.tc ? 4096 : 2048) / u;
  // (partials: not over 1 GiB, unless it takes more for four waves of CTAs, see kMaxPartials)
  const long long per_split = (long long)p->num_seqs * p->num_heads_kv * rows * (p->head_dim + 1) * sizeof(float);
  const long long s_cap = ll_max(ll_max(kMaxPartials / per_split, (4 * slots + ctas - 1) / ctas), 1);
  const long long s_min = ll_min((units + most - 1) / most, s_cap);
  const long long s_max = ll_max(ll_min(ll_min(units / least, s_min + 64), s_cap), s_min);
  w.split_units = (int)most;
  for (long long s = ll_max(s_min, 1), best = -1; s <= s_max; ++s) {
    const long long len = (units + s - 1) / s, waves = (ctas * s + slots - 1) / slots;
    const bool joins = s > 1 && !cluster_fits(w.tc, s, waves);
    const long long cost = waves * (ll_max(len, least) * u + kStartTokens) + (joins ? kJoinTokens : 0);
    if (best < 0 || cost < best) {
      best = cost;
      w.split_units = (int)ll_max(len, least);
    }
  }
  w.max_splits = (int)((units + w.split_units - 1) / w.split_units);
  w.cluster = w.max_splits > 1 && cluster_fits(w.tc, w.max_splits, (ctas * w.max_splits + slots - 1) / slots);
  const size_t parts = w.cluster ? 0 : (size_t)p->num_seqs * p->num_heads_kv * rows * w.max_splits;
  w.part_lse = w.max_splits > 1 ? align256(parts * p->head_dim * sizeof(float)) : 0;
  w.total = w.max_splits > 1 ? w.part_lse + align256(parts * sizeof(float)) : 0;
  return w;
}

static int check(const attn_paged_params_t* p) {
  if (!p || !p->q || !p->key_pool || !p->value_pool || !p->block_table || !p->seq_lengths || !p->out)
    return ATTN_ERR_INVALID;
  if (p->num_seqs <= 0 || p->num_heads_q <= 0 || p->num_heads_kv <= 0 || p->seq_q <= 0 || p->num_blocks <= 0 ||
      p->block_size <= 0 || p->max_blocks_per_seq <= 0 || p->max_context < 0 ||
      p->num_heads_q % p->num_heads_kv != 0)
    return ATTN_ERR_INVALID;
  if (p->num_seqs > 65535) return ATTN_ERR_UNSUPPORTED;  // (a grid dimension)
  if (p->dtype != ATTN_BF16 && p->dtype != ATTN_F16) return ATTN_ERR_UNSUPPORTED;
  if ((p->head_dim != 64 && p->head_dim != 128) || p->block_size % 16 != 0) return ATTN_ERR_UNSUPPORTED;
  if ((long long)p->num_blocks * p->block_size > 0x7fffffffll) return ATTN_ERR_UNSUPPORTED;  // (TMA coordinates)
  if ((long long)p->max_blocks_per_seq * p->block_size > 0x7fffffffll - 4096) return ATTN_ERR_UNSUPPORTED;
  for (const void* x : {p->q, p->key_pool, p->value_pool, (const void*)p->out})
    if (reinterpret_cast<uintptr_t>(x) % 16) return ATTN_ERR_INVALID;
  return ATTN_OK;
}

// Sets a kernel's dynamic shared memory once per device.
template <typename K>
static bool smem_once(K kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const unsigned long long bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load() & bit)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  if (dev < 64) done.fetch_or(bit);
  return true;
}

struct Maps {
  CUtensorMap q, k, v, dk, dv;
};

template <bool BF16, int D, int U, int RW, bool TREE>
static int launch_mma(const Maps& t, const Args& a, cudaStream_t st) {
  using C = MmaCfg<D, U>;
  static std::atomic<unsigned long long> done{0};
  auto kern = rows_mma_kernel<BF16, D, U, RW, TREE>;
  if (!smem_once(kern, C::SMEM, done)) return ATTN_ERR_CUDA;
  const dim3 grid(a.Hkv * a.row_groups, a.max_splits, a.N);
  if (a.cluster) launch_cluster_y(kern, a.max_splits, grid, dim3(kMmaThreads), C::SMEM, st, t.k, t.v, t.dk, t.dv, a);
  else kern<<<grid, kMmaThreads, C::SMEM, st>>>(t.k, t.v, t.dk, t.dv, a);
  return launch_status();
}

template <bool BF16, int D, int NT, bool TREE>
static int launch_tc(const Maps& t, const Args& a, cudaStream_t st) {
  using C = TcCfg<D, NT>;
  static std::atomic<unsigned long long> done{0};
  auto kern = rows_tc_kernel<BF16, D, NT, TREE>;
  // The in-kernel register split draws on exactly C::REGS per thread: with any
  // other launch count the growing warps could wait forever.
  static const bool regs_ok = [&] {
    cudaFuncAttributes fa;
    return cudaFuncGetAttributes(&fa, kern) == cudaSuccess && fa.numRegs == C::REGS;
  }();
  if (!regs_ok) return ATTN_ERR_UNSUPPORTED;
  if (!smem_once(kern, C::SMEM, done)) return ATTN_ERR_CUDA;
  kern<<<dim3(a.Hkv * a.row_groups, a.max_splits, a.N), C::THREADS, C::SMEM, st>>>(t.q, t.k, t.v, t.dk, t.dv, a);
  return launch_status();
}

template <bool BF16, int D, bool TREE>
static int launch_rows(const Plan& w, const Maps& t, const Args& a, cudaStream_t st) {
  int rc;
  if (w.tc)
    rc = a.rows > BM ? launch_tc<BF16, D, 2, TREE>(t, a, st) : launch_tc<BF16, D, 1, TREE>(t, a, st);
  else if (w.unit == 32)
    rc = w.row_tiles == 1 ? launch_mma<BF16, D, 32, 1, TREE>(t, a, st) : launch_mma<BF16, D, 32, 2, TREE>(t, a, st);
  else
    rc = w.row_tiles == 1 ? launch_mma<BF16, D, 16, 1, TREE>(t, a, st) : launch_mma<BF16, D, 16, 2, TREE>(t, a, st);
  if (rc != ATTN_OK || a.max_splits == 1 || a.cluster) return rc;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  launch_overlapped(rows_join_kernel<T, D, TREE>, dim3((a.Hkv * a.rows + 7) / 8, a.N), dim3(256), 0, st, a);
  return launch_status();
}

static int run(const attn_paged_params_t* p, const attn_paged_tree_t* tree, int64_t window, int64_t sinks,
               cudaStream_t st) {
  const Plan w = make_plan(p, tree != nullptr, window, sinks);
  if (w.total > 0 && reinterpret_cast<uintptr_t>(p->workspace) % 16) return ATTN_ERR_INVALID;  // (float4 partials)
  if (w.total > 0 && (!p->workspace || p->workspace_bytes < w.total)) return ATTN_ERR_WORKSPACE;
  if (w.max_splits > 65535) return ATTN_ERR_UNSUPPORTED;
  Maps t;
  const long long tokens = (long long)p->num_blocks * p->block_size;
  if (!make_pool_tmap(&t.k, p->dtype, p->key_pool, tokens, p->num_heads_kv, p->head_dim, w.unit) ||
      !make_pool_tmap(&t.v, p->dtype, p->value_pool, tokens, p->num_heads_kv, p->head_dim, w.unit))
    return ATTN_ERR_INVALID;
  if (tree) {
    if (!make_tmap(&t.dk, p->dtype, tree->draft_keys, p->num_seqs, p->num_heads_kv, p->seq_q, p->head_dim,
                   tree->k_strides, w.span_unit) ||
        !make_tmap(&t.dv, p->dtype, tree->draft_values, p->num_seqs, p->num_heads_kv, p->seq_q, p->head_dim,
                   tree->v_strides, w.span_unit))
      return ATTN_ERR_INVALID;
  } else {
    t.dk = t.k;  // never loaded from
    t.dv = t.v;
  }
  const int rows = p->num_heads_q / p->num_heads_kv * p->seq_q;
  if (w.tc) {
    const int64_t qs[3] = {(int64_t)p->num_heads_kv * rows * p->head_dim, (int64_t)rows * p->head_dim, p->head_dim};
    if (!make_tmap(&t.q, p->dtype, p->q, p->num_seqs, p->num_heads_kv, rows, p->head_dim, qs, BM))
      return ATTN_ERR_INVALID;
  }
  Args a;
  a.N = p->num_seqs; a.Hq = p->num_heads_q; a.Hkv = p->num_heads_kv; a.T = p->seq_q;
  a.group = p->num_heads_q / p->num_heads_kv;
  a.rows = rows;
  a.row_groups = w.row_groups;
  a.BS = p->block_size; a.max_blocks = p->max_blocks_per_seq; a.num_blocks = p->num_blocks;
  a.window = window; a.sinks = sinks;
  a.unit = w.unit; a.span_unit = w.span_unit; a.max_splits = w.max_splits; a.split_units = w.split_units;
  a.cluster = w.cluster;
  a.q = p->q; a.block_table = p->block_table; a.seq_lens = p->seq_lengths;
  a.parents = tree ? tree->parents : nullptr;
  a.tree_lens = tree ? tree->tree_lengths : nullptr;
  a.part_o = reinterpret_cast<float*>(p->workspace);
  a.part_lse = reinterpret_cast<float*>(reinterpret_cast<char*>(p->workspace) + w.part_lse);
  a.out = p->out;
  a.sl2 = p->softmax_scale * kLog2e;
  const bool bf = p->dtype == ATTN_BF16;
  if (p->head_dim == 128) {
    if (tree) return bf ? launch_rows<true, 128, true>(w, t, a, st) : launch_rows<false, 128, true>(w, t, a, st);
    return bf ? launch_rows<true, 128, false>(w, t, a, st) : launch_rows<false, 128, false>(w, t, a, st);
  }
  if (tree) return bf ? launch_rows<true, 64, true>(w, t, a, st) : launch_rows<false, 64, true>(w, t, a, st);
  return bf ? launch_rows<true, 64, false>(w, t, a, st) : launch_rows<false, 64, false>(w, t, a, st);
}

static bool window_ok(int64_t window, int64_t sinks) { return window > 0 && sinks >= 0; }

}  // namespace rows

bool rows_take_status(int* status, int* notice) { return take_status_words(status, notice); }

}  // namespace attnb200

using namespace attnb200;

extern "C" {

size_t attn_paged_window_workspace_size(const attn_paged_params_t* p, int64_t window, int64_t num_sinks) {
  if (rows::check(p) != ATTN_OK || !rows::window_ok(window, num_sinks)) return 0;
  return rows::make_plan(p, false, window, num_sinks).total;
}

int attn_paged_window(const attn_paged_params_t* p, int64_t window, int64_t num_sinks, void* stream) {
  const int rc = rows::check(p);
  if (rc != ATTN_OK) return rc;
  if (!rows::window_ok(window, num_sinks)) return ATTN_ERR_INVALID;
  // (longer than any sequence; keeps the kernels' position arithmetic in range)
  const int64_t far = 1ll << 40;
  return rows::run(p, nullptr, window < far ? window : far, num_sinks < far ? num_sinks : far,
                   reinterpret_cast<cudaStream_t>(stream));
}

size_t attn_paged_tree_workspace_size(const attn_paged_params_t* p) {
  return rows::check(p) == ATTN_OK ? rows::make_plan(p, true, 0, 0).total : 0;
}

int attn_paged_tree(const attn_paged_params_t* p, const attn_paged_tree_t* tree, void* stream) {
  const int rc = rows::check(p);
  if (rc != ATTN_OK) return rc;
  if (!tree || !tree->draft_keys || !tree->draft_values || !tree->parents) return ATTN_ERR_INVALID;
  if (p->seq_q > rows::kMaxTree) return ATTN_ERR_UNSUPPORTED;
  for (const void* x : {tree->draft_keys, tree->draft_values})
    if (reinterpret_cast<uintptr_t>(x) % 16) return ATTN_ERR_INVALID;
  return rows::run(p, tree, 0, 0, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
