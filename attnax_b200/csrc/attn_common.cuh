// Mask semantics shared by every attention kernel.
//
// The flattened mask (attn_mask_t) reproduces the reference's composed
// ScoreMods (attnax/kernels/score_mods.py) and `mask=` argument:
//   causal_mod          keep kv <= q                    (score_mods.py:100-102)
//   sliding_window_mod  keep kv <= q and q - kv < W      (:139-141), or |q-kv| < W (:142)
//   sink_window_mod     keep kv <= q and (q - kv < W or kv < num_sinks); no counterpart in
//                       the reference (first tokens that stay visible to every later query)
//   prefix_lm_mod       keep kv < prefix[b] or kv <= q   (:171-174)
//   document_mask_mod   keep ids[b,q] == ids[b,kv]       (:195-209)
//   alibi_mod           s - slope[h] * |q - kv|          (:76-79)
//   additive_bias_mod   s + bias                         (:235)
//   mask=               where(mask, s, finfo.min)        (attention.py:60-62)
// Dropped scores become -FLT_MAX in the log2 domain (the reference's
// finfo.min), so a row with nothing kept still averages V uniformly; key
// columns past the end of the sequence are -inf and never count.
#pragma once
#include <cfloat>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/attnb200.h"

namespace attnb200 {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

enum TileState : int { kSkip = 0, kPartial = 1, kFull = 2 };

// Tile size of the document-id range tables (both q and kv tiles).
constexpr int kDocTile = 128;

__host__ __device__ inline long long ll_min(long long a, long long b) { return a < b ? a : b; }

// Pool page that block-table entry `e` selects in a pool of `num_blocks`
// pages, read as JAX's array indexing reads pool[block_ids]
// (attnax/paged_cache.py:222-230): a negative entry counts from the end of
// the pool, then the index is clamped into [0, num_blocks).
__host__ __device__ inline long long paged_phys_page(long long e, int num_blocks) {
  if (e < 0) e += num_blocks;
  return e < 0 ? 0 : (e >= num_blocks ? (long long)num_blocks - 1 : e);
}
__host__ __device__ inline long long ll_max(long long a, long long b) { return a > b ? a : b; }

// Classifies the tile [q0,q1) x [k0,k1) of batch b (local positions).
// doc_q_tiles/doc_kv_tiles hold (min,max) ids per kDocTile-row tile; when
// they are null a document mask makes every tile partial.  SINK: the mask
// holds sinks (num_sinks > 0); the instantiations without it never look.
template <bool SINK = false>
__host__ __device__ inline int tile_state(const attn_mask_t& m, const int2* doc_q_tiles,
                                          const int2* doc_kv_tiles, int nq_doc, int nk_doc, int b,
                                          int q0, int q1, int k0, int k1, int bn) {
  int st = kFull;
  if (k1 - k0 < bn) st = kPartial;
  const long long qlo = m.q_offset + q0, qhi = m.q_offset + q1 - 1;
  const long long klo = m.kv_offset + k0, khi = m.kv_offset + k1 - 1;
  if (m.has_band) {
    const long long dmin = qlo - khi, dmax = qhi - klo;
    if (dmax < m.band_lo || (dmin > m.band_hi && !(SINK && klo < m.num_sinks))) return kSkip;
    if (!(dmin >= m.band_lo && (dmax <= m.band_hi || (SINK && khi < m.num_sinks)))) st = kPartial;
  }
  if (m.prefix_len) {
    const long long pref = m.prefix_len[b];
    if (klo >= pref && klo > qhi) return kSkip;
    if (!(khi < pref || khi <= qlo)) st = kPartial;
  }
  if (m.doc_q) {
    // a tile inside one kDocTile tile uses that tile's (min, max) ids (a
    // superset of its own: skip only if disjoint, full only if one document)
    if (doc_q_tiles && doc_kv_tiles && q0 / kDocTile == (q1 - 1) / kDocTile &&
        k0 / kDocTile == (k1 - 1) / kDocTile) {
      const int2 a = doc_q_tiles[(long long)b * nq_doc + q0 / kDocTile];
      const int2 c = doc_kv_tiles[(long long)b * nk_doc + k0 / kDocTile];
      if (a.y < c.x || c.y < a.x) return kSkip;
      if (!(a.x == a.y && c.x == c.y && a.x == c.x)) st = kPartial;
    } else {
      st = kPartial;
    }
  }
  if (m.bool_mask || m.bias) st = kPartial;
  return st;
}

// Local kv-tile index range [lo, hi) that the band allows for rows [q0, q1).
__host__ __device__ inline void band_tile_range(const attn_mask_t& m, int q0, int q1, int seq_kv,
                                                int bn, int* lo, int* hi) {
  const int nk = (seq_kv + bn - 1) / bn;
  *lo = 0;
  *hi = nk;
  if (m.has_band) {
    const long long qlo = m.q_offset + q0, qhi = m.q_offset + q1 - 1;
    long long c_lo = qlo - m.band_hi - m.kv_offset;   // smallest local kv col kept
    long long c_hi = qhi - m.band_lo - m.kv_offset;   // largest
    c_lo = ll_max(c_lo, 0);
    c_hi = ll_min(c_hi, (long long)seq_kv - 1);
    if (c_hi < c_lo) {
      *lo = *hi = 0;
      return;
    }
    *lo = (int)(c_lo / bn);
    *hi = (int)(c_hi / bn) + 1;
  }
}

// Of the band's kv tiles [j_lo, j_hi), those [lo, hi) that rows [q0, q1) keep whole.
__host__ __device__ inline void full_tile_range(const attn_mask_t& m, int q0, int q1, int seq_kv, int bn, int j_lo,
                                                int j_hi, int* lo, int* hi) {
  const long long last = m.q_offset + q0 - m.band_lo - m.kv_offset;        // last column the first row keeps
  const long long first = m.q_offset + q1 - 1 - m.band_hi - m.kv_offset;   // first column the last row keeps
  *lo = first <= 0 ? j_lo : (int)ll_min(ll_max((first + bn - 1) / bn, j_lo), j_hi);
  *hi = last < 0 ? *lo : (int)ll_max(ll_min(ll_min((last + 1) / bn, seq_kv / bn), j_hi), *lo);
}

// kv tiles [0, n) of bn columns that hold a sink some row of [.., q1) may see:
// the last such key is min(num_sinks - 1, q - band_lo) of the last row.
__host__ __device__ inline int sink_tile_count(const attn_mask_t& m, int q1, int seq_kv, int bn) {
  const long long last =
      ll_min(ll_min(m.num_sinks - 1, m.q_offset + q1 - 1 - m.band_lo) - m.kv_offset, (long long)seq_kv - 1);
  return last < 0 ? 0 : (int)(last / bn) + 1;
}

// Of `sink` such tiles, those in front of the band's tiles [j_lo, j_hi) (all, if the band is empty).
__host__ __device__ inline int sink_tiles_before(int sink, int j_lo, int j_hi) {
  return j_hi > j_lo && sink > j_lo ? j_lo : sink;
}

__device__ __forceinline__ float load_bias(const void* p, attn_dtype_t dt, long long idx) {
  if (dt == ATTN_F32) return __ldg(reinterpret_cast<const float*>(p) + idx);
  if (dt == ATTN_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[idx]);
  return __half2float(reinterpret_cast<const __half*>(p)[idx]);
}

// Element transform for one score: raw q.k -> log2-domain score t, with
// every mask and additive term.  `row`/`col` are local positions; with `partial`
// the row must be inside the sequence, a column past its end needs it.  SINK as in
// tile_state: only with num_sinks > 0 (without sinks `kvg < num_sinks` would
// hold for keys at negative positions).
template <bool SINK = false>
__device__ __forceinline__ float mask_score(const attn_mask_t& m, float raw, float sl2,
                                            float slope_l2, int b, int h, int row, int col,
                                            int seq_kv, bool partial) {
  const long long qg = m.q_offset + row, kvg = m.kv_offset + col;
  float t = raw * sl2;
  if (m.alibi_slopes) t -= slope_l2 * fabsf((float)(int)(qg - kvg));
  if (!partial) return t;
  if (col >= seq_kv) return -INFINITY;
  bool keep = true;
  if (m.has_band) {
    const long long d = qg - kvg;
    keep = keep && d >= m.band_lo && (d <= m.band_hi || (SINK && kvg < m.num_sinks));
  }
  if (m.prefix_len) keep = keep && (kvg < (long long)m.prefix_len[b] || kvg <= qg);
  if (m.doc_q)
    keep = keep && (__ldg(m.doc_q + (long long)b * m.doc_q_bstride + qg) ==
                    __ldg(m.doc_kv + (long long)b * m.doc_kv_bstride + kvg));
  if (m.bool_mask)
    keep = keep && m.bool_mask[b * m.mask_strides[0] + h * m.mask_strides[1] +
                               row * m.mask_strides[2] + col * m.mask_strides[3]] != 0;
  if (m.bias)
    t += kLog2e * load_bias(m.bias, m.bias_dtype,
                            b * m.bias_strides[0] + h * m.bias_strides[1] +
                                row * m.bias_strides[2] + col * m.bias_strides[3]);
  return keep ? t : -FLT_MAX;
}

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// What rounding a and b to the 16-bit pair `packed` left of them, rounded to the same type.
template <bool BF16>
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t packed) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&packed);
    const __nv_bfloat162 r = __floats2bfloat162_rn(a - __low2float(h), b - __high2float(h));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 h = *reinterpret_cast<const __half2*>(&packed);
    const __half2 r = __floats2half2_rn(a - __low2float(h), b - __high2float(h));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

// Per-thread constants for transforming one row of a score tile held in
// registers.  Columns are kv positions (forward, dQ) or q positions
// (dK/dV, "transposed").  d(c) = q - kv at column c = d0 + dstep * c.
struct RowCtx {
  float sl2;        // softmax scale * log2(e)
  float slope_l2;   // ALiBi slope * log2(e) (0 when no ALiBi)
  int d0, dstep;
  int ncols;        // columns < ncols are inside the sequence
  int band_lo, band_hi;
  int pref_cols;    // prefix: columns c < pref_cols are kept regardless of d (see make_row_ctx)
  int sink_cols;    // sinks: columns c < sink_cols are kept regardless of band_hi
  int doc_fixed;    // document id of this row
  const int32_t* doc_cols;  // document ids indexed by column
  const uint8_t* bmask;     // bool mask at column 0, column stride bmask_cs
  long long bmask_cs;
  const void* bias;         // bias at column 0, column stride bias_cs
  long long bias_cs;
  attn_dtype_t bias_dtype;
  bool alibi, band, prefix, doc;
};

// Bits e (0..31) of a 32-column chunk with lo <= e <= hi (a keep mask of a
// boundary tile's columns under a band or prefix rule).
__device__ __forceinline__ uint32_t bit_range(long long lo, long long hi) {
  if (hi < 0 || lo > 31 || hi < lo) return 0u;
  const int l = lo < 0 ? 0 : (int)lo, h = hi > 31 ? 31 : (int)hi;
  return (0xffffffffu >> (31 - h)) & (0xffffffffu << l);
}

__device__ __forceinline__ int clamp_i32(long long x) {
  return (int)(x < -(1ll << 30) ? -(1ll << 30) : (x > (1ll << 30) ? (1ll << 30) : x));
}

// row/col0 are local positions of this thread's row and of column 0.  The row
// must be inside the sequence (its document id, mask and bias rows are read);
// rows of a last tile past the end take the last row's, their results are dropped.
// transposed: the row is a kv position and columns are q positions.
__device__ __forceinline__ RowCtx make_row_ctx(const attn_mask_t& m, float sl2, int b, int hq,
                                               int row, int col0, int ncols, bool transposed) {
  RowCtx r;
  r.sl2 = sl2;
  r.alibi = m.alibi_slopes != nullptr;
  r.slope_l2 = r.alibi ? m.alibi_slopes[hq] * kLog2e : 0.f;
  const long long qg0 = m.q_offset + (transposed ? col0 : row);
  const long long kg0 = m.kv_offset + (transposed ? row : col0);
  r.d0 = clamp_i32(qg0 - kg0);
  r.dstep = transposed ? 1 : -1;
  r.ncols = ncols;
  r.band = m.has_band != 0;
  r.band_lo = clamp_i32(m.has_band ? m.band_lo : -(1ll << 40));
  r.band_hi = clamp_i32(m.has_band ? m.band_hi : (1ll << 40));
  // forward columns c < num_sinks - kg0; transposed: all or none
  r.sink_cols = transposed ? (kg0 < m.num_sinks ? (1 << 30) : 0) : clamp_i32(m.num_sinks - kg0);
  r.prefix = m.prefix_len != nullptr;
  r.pref_cols = 0;
  if (r.prefix) {
    const long long pref = m.prefix_len[b];
    // kept when kv < pref: forward columns c < pref - kg0; transposed: all or none
    r.pref_cols = transposed ? (kg0 < pref ? (1 << 30) : 0) : clamp_i32(pref - kg0);
  }
  r.doc = m.doc_q != nullptr;
  r.doc_fixed = 0;
  r.doc_cols = nullptr;
  if (r.doc) {
    if (transposed) {
      r.doc_fixed = m.doc_kv[(long long)b * m.doc_kv_bstride + kg0];
      r.doc_cols = m.doc_q + (long long)b * m.doc_q_bstride + qg0;
    } else {
      r.doc_fixed = m.doc_q[(long long)b * m.doc_q_bstride + qg0];
      r.doc_cols = m.doc_kv + (long long)b * m.doc_kv_bstride + kg0;
    }
  }
  const int qrow = transposed ? col0 : row, kcol = transposed ? row : col0;
  r.bmask = nullptr;
  r.bmask_cs = 0;
  if (m.bool_mask) {
    r.bmask = m.bool_mask + b * m.mask_strides[0] + hq * m.mask_strides[1] +
              (long long)qrow * m.mask_strides[2] + (long long)kcol * m.mask_strides[3];
    r.bmask_cs = transposed ? m.mask_strides[2] : m.mask_strides[3];
  }
  r.bias = nullptr;
  r.bias_cs = 0;
  r.bias_dtype = m.bias_dtype;
  if (m.bias) {
    const long long off = b * m.bias_strides[0] + hq * m.bias_strides[1] +
                          (long long)qrow * m.bias_strides[2] + (long long)kcol * m.bias_strides[3];
    const int es = m.bias_dtype == ATTN_F32 ? 4 : 2;
    r.bias = reinterpret_cast<const char*>(m.bias) + off * es;
    r.bias_cs = transposed ? m.bias_strides[2] : m.bias_strides[3];
  }
  return r;
}

// Raw q.k scores -> log2-domain masked scores, for N register-resident
// columns.  Each feature is its own branch-free unrolled loop so the common
// (full-tile) path stays short.
template <int N, bool SINK = false>
__device__ __forceinline__ void transform_row(float (&s)[N], const RowCtx& r, bool partial) {
  if (r.alibi) {
    const float fd0 = (float)r.d0, fstep = (float)r.dstep;
#pragma unroll
    for (int c = 0; c < N; ++c) s[c] = fmaf(-r.slope_l2, fabsf(fmaf(fstep, (float)c, fd0)), s[c] * r.sl2);
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c) s[c] *= r.sl2;
  }
  if (!partial) return;
  if (r.bias) {
    if (r.bias_dtype == ATTN_F32) {
      const float* p = reinterpret_cast<const float*>(r.bias);
#pragma unroll
      for (int c = 0; c < N; ++c)
        if (c < r.ncols) s[c] = fmaf(kLog2e, __ldg(p + c * r.bias_cs), s[c]);
    } else {
#pragma unroll
      for (int c = 0; c < N; ++c)
        if (c < r.ncols) s[c] = fmaf(kLog2e, load_bias(r.bias, r.bias_dtype, c * r.bias_cs), s[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const int d = r.d0 + r.dstep * c;
    bool keep = !r.band || (d >= r.band_lo && (d <= r.band_hi || (SINK && c < r.sink_cols)));
    if (r.prefix) keep = keep && (c < r.pref_cols || d >= 0);
    s[c] = c < r.ncols ? (keep ? s[c] : -FLT_MAX) : -INFINITY;
  }
  if (r.doc) {
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < r.ncols && __ldg(r.doc_cols + c) != r.doc_fixed) s[c] = -FLT_MAX;
  }
  if (r.bmask) {
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < r.ncols && r.bmask[c * r.bmask_cs] == 0) s[c] = -FLT_MAX;
  }
}

}  // namespace attnb200
