// Tile tables of a document mask: id ranges per tile, the tiles that can meet, and the launch order.
#pragma once
#include "attn_common.cuh"

namespace attnb200 {

// For every row tile t (of batch b): the range [lo, hi) of column tiles
// whose (min, max) id range overlaps row tile t's, from the per-tile ranges
// of doc_tile_range_kernel -- exact for sorted ids (packed documents), a
// superset otherwise.  One warp per row tile.
__global__ void doc_cross_range_kernel(const int2* row_tiles, int n_row, const int2* col_tiles, int n_col,
                                       int2* out) {
  const int t = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32, lane = threadIdx.x & 31;
  const int b = blockIdx.y;
  if (t >= n_row) return;
  const int2 r = row_tiles[(long long)b * n_row + t];
  int lo = 0x7fffffff, hi = -1;
  for (int c = lane; c < n_col; c += 32) {
    const int2 k = col_tiles[(long long)b * n_col + c];
    if (!(r.y < k.x || k.y < r.x)) {
      lo = min(lo, c);
      hi = max(hi, c);
    }
  }
  for (int o = 16; o > 0; o >>= 1) {
    lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (lane == 0) out[(long long)b * n_row + t] = hi < 0 ? make_int2(0, 0) : make_int2(lo, hi + 1);
}

// Launch order of the forward's two-query-tile CTAs under a document mask.
// Per batch, CTA indices are ranked by their kv-tile count (the document
// range of q_jr intersected with the band, summed over the CTA's two query
// tiles of bm == kDocTile rows), largest first, later tiles first on ties,
// so the longest CTAs start in the first wave.  One block per batch;
// n_ctas ints of dynamic shared memory.
__global__ void doc_cta_order_kernel(attn_mask_t m, const int2* q_jr, int nq_doc, int seq_q, int seq_kv, int bm,
                                     int bn, int n_ctas, int* order) {
  extern __shared__ int work[];
  const int b = blockIdx.x;
  for (int c = threadIdx.x; c < n_ctas; c += blockDim.x) {
    int tot = 0;
    for (int x = 0; x < 2; ++x) {
      const int q0 = c * 2 * bm + x * bm;
      if (q0 >= seq_q) continue;
      int lo, hi;
      band_tile_range(m, q0, min(q0 + bm, seq_q), seq_kv, bn, &lo, &hi);
      const int2 r = q_jr[(long long)b * nq_doc + q0 / kDocTile];
      tot += max(0, min(hi, r.y) - max(lo, r.x));
    }
    work[c] = tot;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < n_ctas; c += blockDim.x) {
    const int wc = work[c];
    int rank = 0;
    for (int o = 0; o < n_ctas; ++o) rank += (work[o] > wc) || (work[o] == wc && o > c);
    order[(long long)b * n_ctas + rank] = c;
  }
}

// (min, max) of document ids over kDocTile-row tiles of global positions
// offset + [t*kDocTile, min((t+1)*kDocTile, len)).
__global__ void doc_tile_range_kernel(const int32_t* ids, long long bstride, long long offset,
                                      int len, int ntiles, int2* out) {
  const int t = blockIdx.x, b = blockIdx.y;
  int lo = 0x7fffffff, hi = -0x7fffffff - 1;
  for (int i = t * kDocTile + threadIdx.x; i < min((t + 1) * kDocTile, len); i += blockDim.x) {
    const int v = ids[(long long)b * bstride + offset + i];
    lo = min(lo, v);
    hi = max(hi, v);
  }
  for (int o = 16; o > 0; o >>= 1) {
    lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  __shared__ int slo[32], shi[32];
  const int w = threadIdx.x / 32;
  if ((threadIdx.x & 31) == 0) {
    slo[w] = lo;
    shi[w] = hi;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < (int)blockDim.x / 32; ++i) {
      lo = min(lo, slo[i]);
      hi = max(hi, shi[i]);
    }
    out[(long long)b * ntiles + t] = make_int2(lo, hi);
  }
}

}  // namespace attnb200
