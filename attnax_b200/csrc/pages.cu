// Page operators of the paged KV cache: copying, forking, freeing and
// compacting pages, and appending accepted drafts, for whole batches without a
// host round trip.  Sets of pages are bit maps (one bit per page of the pool);
// lists come out in ascending order, so results do not depend on the order in
// which CTAs run.  The bytes moved bound the copies; the rest is launch and
// memory latency.
#include <cooperative_groups.h>

#include <atomic>
#include <climits>

#include "attn_common.cuh"
#include "host_util.h"
#include "sm100.cuh"

namespace attnb200 {
namespace pages {

__device__ __forceinline__ void skip_notice() { atomicCAS(&g_notice, 0, kNoticePageList); }

// Copies `n` vectors by the whole block, kUnroll loads in flight per thread.
template <typename V>
__device__ __forceinline__ void copy_vecs(const V* __restrict__ src, V* __restrict__ dst, long long n) {
  constexpr int kUnroll = 8;
  const int step = blockDim.x;
  long long i = threadIdx.x;
  for (; i + (kUnroll - 1) * (long long)step < n; i += kUnroll * (long long)step) {
    V v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = __ldcs(src + i + u * step);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) __stcs(dst + i + u * step, v[u]);
  }
  for (; i < n; i += step) dst[i] = src[i];
}

struct Pool {
  void *k, *v;
  int num_blocks;
  long long vecs;  // vectors per page
  float *ks, *vs;  // pools of 8-bit codes: heads scales per page, or null
  int heads;
};

__device__ __forceinline__ void copy_scales(const Pool& p, float* scales, int src, int dst) {
  if (!scales) return;
  for (int h = threadIdx.x; h < p.heads; h += blockDim.x)
    scales[(long long)dst * p.heads + h] = scales[(long long)src * p.heads + h];
}

template <typename V>
__device__ __forceinline__ void copy_page(const Pool& p, int src, int dst) {
  copy_vecs(reinterpret_cast<const V*>(p.k) + src * p.vecs, reinterpret_cast<V*>(p.k) + dst * p.vecs, p.vecs);
  copy_vecs(reinterpret_cast<const V*>(p.v) + src * p.vecs, reinterpret_cast<V*>(p.v) + dst * p.vecs, p.vecs);
  copy_scales(p, p.ks, src, dst);
  copy_scales(p, p.vs, src, dst);
}

// ------------------------------------------------------------------- copy --
// One CTA per E entries and pool.  It looks through both lists itself, so no
// pass over the lists and no scratch is needed; with many entries E of them
// share that pass (2048 entries of 32 KB pages: 47.2 us one by one).
template <typename V, int E>
__global__ void __launch_bounds__(256) copy_kernel(Pool p, const int32_t* src, const int32_t* dst, int n) {
  const int i0 = blockIdx.x * E;
  int s[E], d[E];
  uint32_t bad = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool in = i0 + e < n;
    s[e] = in ? src[i0 + e] : 0;
    d[e] = in ? dst[i0 + e] : 0;
    if (s[e] < 0 || s[e] >= p.num_blocks || d[e] < 0 || d[e] >= p.num_blocks) bad |= 1u << e;
  }
  for (int j = threadIdx.x; j < n; j += 256) {
    const int sj = src[j], dj = dst[j];
#pragma unroll
    for (int e = 0; e < E; ++e)
      if ((j < i0 + e && dj == d[e]) || (j != i0 + e && sj == d[e])) bad |= 1u << e;
  }
  V* pool = reinterpret_cast<V*>(blockIdx.y ? p.v : p.k);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool skip = __syncthreads_or((bad >> e) & 1u);
    if (i0 + e >= n || (s[e] == d[e] && s[e] >= 0 && s[e] < p.num_blocks)) continue;
    if (skip) {
      if (threadIdx.x == 0) skip_notice();
    } else {
      copy_vecs(pool + s[e] * p.vecs, pool + d[e] * p.vecs, p.vecs);
      copy_scales(p, blockIdx.y ? p.vs : p.ks, s[e], d[e]);
    }
  }
}

// ------------------------------------------------------------------- fork --
struct ForkArgs {
  const int32_t *table, *lens, *src, *dst, *free_ids;
  int num_seqs, max_blocks, block_size, n, num_free;
  int32_t *table_out, *lens_out, *used;
};

__device__ __forceinline__ bool in_range(int x, int n) { return x >= 0 && x < n; }

// Whether fork j takes a page of free_ids: its source's last page is not full.
__device__ __forceinline__ bool takes_page(const ForkArgs& a, int j) {
  const int s = a.src[j];
  if (!in_range(s, a.num_seqs) || !in_range(a.dst[j], a.num_seqs)) return false;
  const int len = max(a.lens[s], 0);
  return len % a.block_size != 0 && len / a.block_size < a.max_blocks;
}

// CTAs [0, num_seqs): rows that no fork replaces.  CTA num_seqs + i: fork i.
template <typename V>
__global__ void __launch_bounds__(256) fork_kernel(Pool p, ForkArgs a) {
  const int i = (int)blockIdx.x - a.num_seqs;
  if (i < 0) {
    const int r = blockIdx.x;
    bool replaced = false;
    for (int j = threadIdx.x; j < a.n; j += blockDim.x)
      replaced = replaced || (a.dst[j] == r && in_range(a.src[j], a.num_seqs));
    if (__syncthreads_or(replaced)) return;
    for (int c = threadIdx.x; c < a.max_blocks; c += blockDim.x)
      a.table_out[(long long)r * a.max_blocks + c] = a.table[(long long)r * a.max_blocks + c];
    if (threadIdx.x == 0) a.lens_out[r] = a.lens[r];
    return;
  }
  // free_ids taken by the forks in front of this one, and by all (the last CTA reports them)
  int before = 0;
  bool twice = false;
  for (int j = threadIdx.x; j < i; j += blockDim.x) {
    before += takes_page(a, j);
    twice = twice || (a.dst[j] == a.dst[i] && in_range(a.src[j], a.num_seqs));
  }
  __shared__ int sum;
  if (threadIdx.x == 0) sum = 0;
  __syncthreads();
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if ((threadIdx.x & 31) == 0 && before) atomicAdd(&sum, before);
  twice = __syncthreads_or(twice);
  const int k = sum;
  const bool takes = takes_page(a, i);
  // (a fork that is skipped below has taken its id all the same: the ids go by the list alone)
  if (i == a.n - 1 && threadIdx.x == 0) *a.used = min(k + (takes ? 1 : 0), a.num_free);
  const int s = a.src[i], d = a.dst[i];
  if (!in_range(s, a.num_seqs) || !in_range(d, a.num_seqs) || twice) {
    if (threadIdx.x == 0) skip_notice();
    return;
  }
  const int len = max(a.lens[s], 0);
  const int cols = min((len + a.block_size - 1) / a.block_size, a.max_blocks);
  const int32_t* row = a.table + (long long)s * a.max_blocks;
  int32_t* out = a.table_out + (long long)d * a.max_blocks;
  int fresh = -1, tail = -1;
  if (takes) {
    tail = row[cols - 1];
    fresh = k < a.num_free ? a.free_ids[k] : -1;
    bool taken = false;  // an id listed twice is the first one's
    for (int j = threadIdx.x; j < min(k, a.num_free); j += blockDim.x) taken = taken || a.free_ids[j] == fresh;
    if (__syncthreads_or(taken) || !in_range(fresh, p.num_blocks) || !in_range(tail, p.num_blocks)) {
      // no page for the copy: the row keeps its full pages and their tokens
      if (threadIdx.x == 0) skip_notice();
      fresh = -1;
    }
  }
  const int keep = takes && fresh < 0 ? cols - 1 : cols;
  for (int c = threadIdx.x; c < a.max_blocks; c += blockDim.x)
    out[c] = c < keep ? (takes && c == cols - 1 ? fresh : row[c]) : -1;
  if (threadIdx.x == 0) a.lens_out[d] = takes && fresh < 0 ? keep * a.block_size : len;
  if (fresh >= 0 && fresh != tail) copy_page<V>(p, tail, fresh);
}

// ------------------------------------------------------------------- sets --
// Sets page bit e of a map (entries outside the pool refer to nothing).
__device__ __forceinline__ void set_bit(uint32_t* map, int e, int num_blocks) {
  if (e >= 0 && e < num_blocks) atomicOr(map + (e >> 5), 1u << (e & 31));
}

// Exclusive sum of x over the 1024 threads of a block; *total the sum.
__device__ __forceinline__ int block_scan(int x, int* total) {
  __shared__ int warp_sum[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int v = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();
  if (lane == 31) warp_sum[warp] = v;
  __syncthreads();
  int w = warp_sum[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  const int base = warp > 0 ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
  return base + v - x;
}

struct FreeArgs {
  const int32_t *table, *lens, *seqs;
  int num_seqs, max_blocks, block_size, num_blocks, n;
  long long window, sinks;  // window > 0: free_window
  int32_t *table_out, *lens_out, *freed, *count;
  uint32_t *live, *gone;
};

// Whether page column c of a row goes (free_window); `lo`: first key in the window of the query at its length.
__device__ __forceinline__ bool out_of_window(const FreeArgs& a, long long lo, int c) {
  return (long long)(c + 1) * a.block_size <= lo && (long long)c * a.block_size >= a.sinks;
}

// ---- sets of up to kClusterPages pages: one cluster, bit maps in shared memory ----
// Eight CTAs mark a share of the table each in maps of their own; each then
// joins one eighth of the words of all maps through distributed shared memory
// and writes that part of the list.  One launch in place of clearing, marking
// and listing (64 rows of 256 columns, 16000 pages: 12 us and 16 us of kernels
// before, for free and compact).
namespace cg = cooperative_groups;
constexpr int kCluster = 8;
constexpr int kClusterPages = 800 * 1024;  // two maps: 200 KB of shared memory
constexpr int kChunk = 256;                // table columns a warp marks at a time

// Joins words [lo, hi) of every CTA's map `bits` into this CTA's own.
__device__ __forceinline__ void join_maps(cg::cluster_group& cl, uint32_t* bits, int lo, int hi) {
  for (int w = lo + threadIdx.x; w < hi; w += 1024) {
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < kCluster; ++r) m |= cl.map_shared_rank(bits, r)[w];
    bits[w] = m;  // (no other CTA reads this CTA's copy of its own words)
  }
}

// Sum of x over the CTAs in front of this one, and over all; x is block-uniform.
__device__ __forceinline__ int cluster_scan(cg::cluster_group& cl, int* slot, int x, int* total) {
  if (threadIdx.x == 0) *slot = x;
  cl.sync();
  int before = 0, all = 0;
#pragma unroll
  for (int r = 0; r < kCluster; ++r) {
    const int v = *cl.map_shared_rank(slot, r);
    before += r < (int)blockIdx.x ? v : 0;
    all += v;
  }
  *total = all;
  return before;
}

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(1024) free_cluster_kernel(FreeArgs a) {
  extern __shared__ uint32_t maps[];
  __shared__ int slot;
  cg::cluster_group cl = cg::this_cluster();
  const int words = (a.num_blocks + 31) / 32, per = (words + kCluster - 1) / kCluster;
  uint32_t *live = maps, *gone = maps + words;
  for (int w = threadIdx.x; w < 2 * words; w += 1024) maps[w] = 0u;
  __syncthreads();
  const int warp = blockIdx.x + kCluster * (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int chunks = (a.max_blocks + kChunk - 1) / kChunk;
  for (long long it = warp; it < (long long)a.num_seqs * chunks; it += kCluster * 32) {
    const int r = (int)(it / chunks), c0 = (int)(it % chunks) * kChunk;
    const int len = max(a.lens[r], 0);
    bool ends = false;
    if (a.window <= 0) {
      for (int j = lane; j < a.n; j += 32) {
        ends = ends || a.seqs[j] == r;
        if (it == 0 && !(a.seqs[j] >= 0 && a.seqs[j] < a.num_seqs)) skip_notice();
      }
      ends = __any_sync(0xffffffffu, ends);
      if (lane == 0 && c0 == 0) a.lens_out[r] = ends ? 0 : a.lens[r];
    }
    const long long lo = len - a.window + 1;
#pragma unroll
    for (int u = 0; u < kChunk / 32; ++u) {
      const int c = c0 + u * 32 + lane;
      if (c >= a.max_blocks) continue;
      const long long at = (long long)r * a.max_blocks + c;
      const int e = a.table[at];
      const bool out = a.window > 0 ? out_of_window(a, lo, c) : ends;
      a.table_out[at] = out ? -1 : e;
      set_bit(out ? gone : live, e, a.num_blocks);
    }
  }
  cl.sync();
  const int lo = min((int)blockIdx.x * per, words), hi = min(lo + per, words);
  join_maps(cl, live, lo, hi);
  join_maps(cl, gone, lo, hi);
  int mine = 0, total, all;
  for (int w = lo + threadIdx.x; w < hi; w += 1024) mine += __popc(gone[w] & ~live[w]);
  block_scan(mine, &total);
  int base = cluster_scan(cl, &slot, total, &all);
  for (int w0 = lo; w0 < hi; w0 += 1024) {
    const int w = w0 + threadIdx.x;
    uint32_t m = w < hi ? gone[w] & ~live[w] : 0u;
    int at = base + block_scan(__popc(m), &total);
    for (; m; m &= m - 1) a.freed[at++] = w * 32 + __ffs(m) - 1;
    base += total;
  }
  for (long long i = (long long)all + blockIdx.x * 1024 + threadIdx.x; i < a.num_blocks; i += kCluster * 1024)
    a.freed[i] = -1;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.count = all;
  cl.sync();  // (the others have read this CTA's sum)
}

// ---- larger pools: maps in the workspace ----
// One CTA per row: the new row, and the page sets of what goes and what stays.
__global__ void __launch_bounds__(256) free_mark_kernel(FreeArgs a) {
  const int r = blockIdx.x, len = max(a.lens[r], 0);
  bool ends = false;
  if (a.window <= 0) {
    for (int j = threadIdx.x; j < a.n; j += blockDim.x) {
      ends = ends || a.seqs[j] == r;
      if (r == 0 && !(a.seqs[j] >= 0 && a.seqs[j] < a.num_seqs)) skip_notice();
    }
    ends = __syncthreads_or(ends);
    if (threadIdx.x == 0) a.lens_out[r] = ends ? 0 : a.lens[r];
  }
  const long long lo = len - a.window + 1;  // first key in the window of the query at position len
  for (int c = threadIdx.x; c < a.max_blocks; c += blockDim.x) {
    const long long at = (long long)r * a.max_blocks + c;
    const int e = a.table[at];
    const bool out = a.window > 0 ? out_of_window(a, lo, c) : ends;
    a.table_out[at] = out ? -1 : e;
    set_bit(out ? a.gone : a.live, e, a.num_blocks);
  }
}

// Lists the pages that are gone and not live, ascending.  One block.
__global__ void __launch_bounds__(1024) free_list_kernel(FreeArgs a) {
  const int words = (a.num_blocks + 31) / 32;
  int base = 0;
  for (int w0 = 0; w0 < words; w0 += 1024) {
    const int w = w0 + threadIdx.x;
    uint32_t m = w < words ? a.gone[w] & ~a.live[w] : 0u;
    int total;
    int at = base + block_scan(__popc(m), &total);
    for (; m; m &= m - 1) a.freed[at++] = w * 32 + __ffs(m) - 1;
    base += total;
  }
  for (int i = base + threadIdx.x; i < a.num_blocks; i += blockDim.x) a.freed[i] = -1;
  if (threadIdx.x == 0) *a.count = base;
}

struct CompactArgs {
  const int32_t* table;
  long long entries;
  int num_blocks;
  int32_t *table_out, *num_live;
  uint32_t* live;
  int32_t *holes, *movers, *rank;  // hole k, moved page k, and k of a moved page
  int32_t* moves;                  // number of moves
};

// Pages of word w below n_live, as a mask.
__device__ __forceinline__ uint32_t pages_below(int w, int n_live) {
  const int below = max(0, min(32, n_live - w * 32));
  return below >= 32 ? 0xffffffffu : (1u << below) - 1u;
}

// One cluster, as free_cluster_kernel.
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(1024) compact_cluster_kernel(CompactArgs a) {
  extern __shared__ uint32_t live[];
  __shared__ int slot[3];
  cg::cluster_group cl = cg::this_cluster();
  pdl_launch_next();
  const int words = (a.num_blocks + 31) / 32, per = (words + kCluster - 1) / kCluster;
  for (int w = threadIdx.x; w < words; w += 1024) live[w] = 0u;
  __syncthreads();
#pragma unroll 4
  for (long long i = blockIdx.x * 1024ll + threadIdx.x; i < a.entries; i += kCluster * 1024)
    set_bit(live, a.table[i], a.num_blocks);
  cl.sync();
  const int lo = min((int)blockIdx.x * per, words), hi = min(lo + per, words);
  join_maps(cl, live, lo, hi);
  int mine = 0, total, n_live, moves;
  for (int w = lo + threadIdx.x; w < hi; w += 1024) mine += __popc(live[w]);
  block_scan(mine, &total);
  const int live_before = cluster_scan(cl, &slot[0], total, &n_live);
  mine = 0;
  for (int w = lo + threadIdx.x; w < hi; w += 1024) mine += __popc(live[w] & ~pages_below(w, n_live));
  block_scan(mine, &total);
  int movers = cluster_scan(cl, &slot[1], total, &moves);
  // holes in front of this share: its first page less the live pages below it (no holes behind n_live)
  int holes = lo * 32 - live_before;
  for (int w0 = lo; w0 < hi; w0 += 1024) {
    const int w = w0 + threadIdx.x;
    const uint32_t l = w < hi ? live[w] : 0u, low = pages_below(w, n_live);
    uint32_t h = w < hi ? ~l & low : 0u, m = l & ~low;
    int at = holes + block_scan(__popc(h), &total);
    holes += total;
    for (; h; h &= h - 1) a.holes[at++] = w * 32 + __ffs(h) - 1;
    at = movers + block_scan(__popc(m), &total);
    movers += total;
    for (; m; m &= m - 1, ++at) {
      const int page = w * 32 + __ffs(m) - 1;
      a.movers[at] = page;
      a.rank[page] = at;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *a.num_live = n_live;
    *a.moves = moves;
  }
  cl.sync();  // (the others have read this CTA's sums)
}

__global__ void __launch_bounds__(256) compact_mark_kernel(CompactArgs a) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < a.entries; i += gridDim.x * 256ll)
    set_bit(a.live, a.table[i], a.num_blocks);
}

// Live pages at or past their number, and the holes below it, both ascending.  One block.
__global__ void __launch_bounds__(1024) compact_list_kernel(CompactArgs a) {
  const int words = (a.num_blocks + 31) / 32;
  int mine = 0, n_live = 0;
  for (int w = threadIdx.x; w < words; w += 1024) mine += __popc(a.live[w]);
  block_scan(mine, &n_live);
  int holes = 0, movers = 0;
  for (int w0 = 0; w0 < words; w0 += 1024) {
    const int w = w0 + threadIdx.x;
    const uint32_t l = w < words ? a.live[w] : 0u;
    const uint32_t low = pages_below(w, n_live);
    uint32_t h = w < words ? ~l & low : 0u, m = l & ~low;
    int total;
    int at = holes + block_scan(__popc(h), &total);
    holes += total;
    for (; h; h &= h - 1) a.holes[at++] = w * 32 + __ffs(h) - 1;
    at = movers + block_scan(__popc(m), &total);
    movers += total;
    for (; m; m &= m - 1, ++at) {
      const int page = w * 32 + __ffs(m) - 1;
      a.movers[at] = page;
      a.rank[page] = at;
    }
  }
  if (threadIdx.x == 0) {
    *a.num_live = n_live;
    *a.moves = movers;  // (as many as holes)
  }
}

// CTAs [0, copiers) move pages; the others write the table's new entries.
template <typename V>
__global__ void __launch_bounds__(256) compact_move_kernel(Pool p, CompactArgs a, int copiers) {
  pdl_wait_previous();
  if ((int)blockIdx.x < copiers) {
    const int n = *a.moves;
    for (int i = blockIdx.x; i < n; i += copiers) copy_page<V>(p, a.movers[i], a.holes[i]);
    return;
  }
  const int n_live = *a.num_live;
  const long long step = (long long)(gridDim.x - copiers) * 256;
  for (long long i = ((int)blockIdx.x - copiers) * 256ll + threadIdx.x; i < a.entries; i += step) {
    const int e = a.table[i];
    a.table_out[i] = e >= n_live && e < a.num_blocks ? a.holes[a.rank[e]] : e;
  }
}

// ----------------------------------------------------------------- accept --
struct AcceptArgs {
  const int32_t *table, *lens, *accepted, *acc_lens;
  int num_seqs, max_blocks, num_blocks, block_size, heads, row_vecs;  // vectors of one head's row
  int drafts, max_acc;
  const void *dk, *dv;
  long long ks[3], vs[3];  // in vectors
  void *k, *v;
  int32_t *lens_out, *bad;
};

// Pool row of accepted token i of sequence s and its draft, or false.
__device__ __forceinline__ bool accept_at(const AcceptArgs& a, int s, int i, long long* row, int* tok) {
  const int pos = a.lens[s] + i, col = pos / a.block_size;
  *tok = a.accepted[(long long)s * a.max_acc + i];
  if (pos < 0 || col >= a.max_blocks || !in_range(*tok, a.drafts)) return false;
  const int page = a.table[(long long)s * a.max_blocks + col];
  *row = (long long)page * a.block_size + pos % a.block_size;
  return in_range(page, a.num_blocks);
}

__global__ void accept_check_kernel(AcceptArgs a) {
  const int s = blockIdx.x, n = a.acc_lens[s];
  bool bad = n < 0 || n > a.max_acc;
  for (int i = threadIdx.x; i < min(n, a.max_acc); i += blockDim.x) {
    long long row;
    int tok;
    bad = bad || !accept_at(a, s, i, &row, &tok);
  }
  if (bad) atomicMin(a.bad, s);
}

template <typename V>
__global__ void __launch_bounds__(256) accept_kernel(AcceptArgs a) {
  const int s = blockIdx.y, n = min(max(a.acc_lens[s], 0), a.max_acc);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.lens_out[s] = a.lens[s] + n;
    if (n != a.acc_lens[s]) skip_notice();
  }
  const int per_tok = a.heads * a.row_vecs;
  const int x = blockIdx.x * 256 + threadIdx.x;
  const int i = x / per_tok;
  if (i >= n) return;
  const int h = x % per_tok / a.row_vecs, e = x % a.row_vecs;
  long long row;
  int tok;
  if (!accept_at(a, s, i, &row, &tok)) {
    skip_notice();
    return;
  }
  const long long dst = row * per_tok + h * a.row_vecs + e;
  reinterpret_cast<V*>(a.k)[dst] =
      reinterpret_cast<const V*>(a.dk)[s * a.ks[0] + h * a.ks[1] + tok * a.ks[2] + e];
  reinterpret_cast<V*>(a.v)[dst] =
      reinterpret_cast<const V*>(a.dv)[s * a.vs[0] + h * a.vs[1] + tok * a.vs[2] + e];
}

// ------------------------------------------------------------------- host --
// Whether the pools hold 8-bit codes.
static bool codes(const attn_paged_cache_t* c) {
  return (int)c->dtype == ATTN_POOL_E4M3 || (int)c->dtype == ATTN_POOL_INT8;
}

static bool cache_ok(const attn_paged_cache_t* c, bool pools, bool table) {
  if (!c || c->num_blocks <= 0 || c->block_size <= 0 || c->num_heads_kv <= 0 || c->head_dim <= 0) return false;
  if (c->dtype != ATTN_F32 && c->dtype != ATTN_BF16 && c->dtype != ATTN_F16 && !codes(c)) return false;
  if (pools && (!c->key_pool || !c->value_pool || (codes(c) && (!c->key_scales || !c->value_scales)))) return false;
  return !table || (c->num_seqs > 0 && c->max_blocks_per_seq > 0 && c->block_table && c->seq_lengths);
}

// Widest vector that divides `bytes` and fits the alignment of the addresses in `bits`.
static int vec_bytes(long long bytes, uintptr_t bits) {
  int v = 16;
  while (v > 1 && (bytes % v || bits % v)) v /= 2;
  return v;
}

static uintptr_t addr(const void* p) { return reinterpret_cast<uintptr_t>(p); }

static Pool make_pool(const attn_paged_cache_t* c, int* vec) {
  const long long bytes =
      (long long)c->block_size * c->num_heads_kv * c->head_dim * (codes(c) ? 1 : dtype_size(c->dtype));
  *vec = vec_bytes(bytes, addr(c->key_pool) | addr(c->value_pool));
  return Pool{c->key_pool, c->value_pool, c->num_blocks, bytes / *vec,
              codes(c) ? c->key_scales : nullptr, codes(c) ? c->value_scales : nullptr, c->num_heads_kv};
}

#define PAGES_BY_VEC(vec, CALL) \
  do {                          \
    if (vec == 16) CALL(uint4); \
    else if (vec == 8) CALL(uint2); \
    else if (vec == 4) CALL(uint32_t); \
    else if (vec == 2) CALL(uint16_t); \
    else CALL(uint8_t);         \
  } while (0)

static size_t map_bytes(const attn_paged_cache_t* c) { return align256((size_t)(c->num_blocks + 31) / 32 * 4); }

// Sets a cluster kernel's dynamic shared memory (the most it can need) once per device.
template <typename K>
static bool cluster_smem(K kernel, int maps, std::atomic<unsigned long long>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const unsigned long long bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load() & bit)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, maps * kClusterPages / 8) !=
      cudaSuccess)
    return false;
  if (dev < 64) done.fetch_or(bit);
  return true;
}

static int free_pages(const attn_paged_cache_t* c, FreeArgs a, void* workspace, size_t bytes, cudaStream_t st) {
  a.table = c->block_table; a.lens = c->seq_lengths;
  a.num_seqs = c->num_seqs; a.max_blocks = c->max_blocks_per_seq;
  a.block_size = c->block_size; a.num_blocks = c->num_blocks;
  if (c->num_blocks <= kClusterPages) {
    static std::atomic<unsigned long long> done{0};
    if (!cluster_smem(free_cluster_kernel, 2, done)) return ATTN_ERR_CUDA;
    free_cluster_kernel<<<kCluster, 1024, 2 * ((c->num_blocks + 31) / 32) * 4, st>>>(a);
    return launch_status();
  }
  const size_t need = 2 * map_bytes(c);
  if (addr(workspace) % 4) return ATTN_ERR_INVALID;
  if (!workspace || bytes < need) return ATTN_ERR_WORKSPACE;
  if (cudaMemsetAsync(workspace, 0, need, st) != cudaSuccess) return ATTN_ERR_CUDA;
  a.live = reinterpret_cast<uint32_t*>(workspace);
  a.gone = reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(workspace) + map_bytes(c));
  free_mark_kernel<<<c->num_seqs, 256, 0, st>>>(a);
  free_list_kernel<<<1, 1024, 0, st>>>(a);
  return launch_status(2);
}

}  // namespace pages

bool pages_take_status(int* status, int* notice) { return take_status_words(status, notice); }

}  // namespace attnb200

using namespace attnb200;

extern "C" {

int attn_paged_copy(const attn_paged_cache_t* c, const int32_t* src, const int32_t* dst, int32_t n, void* stream) {
  if (!pages::cache_ok(c, true, false) || n < 0) return ATTN_ERR_INVALID;
  if (n == 0) return ATTN_OK;
  if (!src || !dst) return ATTN_ERR_INVALID;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int vec;
  const pages::Pool p = pages::make_pool(c, &vec);
  const bool many = n >= 1024;
#define CALL(V) \
  (many ? pages::copy_kernel<V, 4><<<dim3((n + 3) / 4, 2), 256, 0, st>>>(p, src, dst, n) \
        : pages::copy_kernel<V, 1><<<dim3(n, 2), 256, 0, st>>>(p, src, dst, n))
  PAGES_BY_VEC(vec, CALL);
#undef CALL
  return launch_status();
}

int attn_paged_fork(const attn_paged_cache_t* c, const int32_t* src, const int32_t* dst, int32_t n,
                    const int32_t* free_ids, int32_t num_free, int32_t* table_out, int32_t* lengths_out,
                    int32_t* used, void* stream) {
  if (!pages::cache_ok(c, true, true) || n <= 0 || num_free < 0 || (num_free > 0 && !free_ids) || !src || !dst ||
      !table_out || !lengths_out || !used || table_out == c->block_table || lengths_out == c->seq_lengths)
    return ATTN_ERR_INVALID;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int vec;
  const pages::Pool p = pages::make_pool(c, &vec);
  const pages::ForkArgs a{c->block_table, c->seq_lengths, src, dst, free_ids, c->num_seqs, c->max_blocks_per_seq,
                          c->block_size, n, num_free, table_out, lengths_out, used};
#define CALL(V) pages::fork_kernel<V><<<c->num_seqs + n, 256, 0, st>>>(p, a)
  PAGES_BY_VEC(vec, CALL);
#undef CALL
  return launch_status();
}

size_t attn_paged_free_workspace_size(const attn_paged_cache_t* c) {
  return pages::cache_ok(c, false, false) && c->num_blocks > pages::kClusterPages ? 2 * pages::map_bytes(c) : 0;
}

int attn_paged_free(const attn_paged_cache_t* c, const int32_t* seqs, int32_t n, int32_t* table_out,
                    int32_t* lengths_out, int32_t* freed, int32_t* count, void* workspace, size_t workspace_bytes,
                    void* stream) {
  if (!pages::cache_ok(c, false, true) || n < 0 || (n > 0 && !seqs) || !table_out || !lengths_out || !freed || !count)
    return ATTN_ERR_INVALID;
  pages::FreeArgs a{};
  a.seqs = seqs; a.n = n;
  a.table_out = table_out; a.lens_out = lengths_out; a.freed = freed; a.count = count;
  return pages::free_pages(c, a, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

int attn_paged_free_window(const attn_paged_cache_t* c, int64_t window, int64_t num_sinks, int32_t* table_out,
                           int32_t* freed, int32_t* count, void* workspace, size_t workspace_bytes, void* stream) {
  if (!pages::cache_ok(c, false, true) || window <= 0 || num_sinks < 0 || !table_out || !freed || !count)
    return ATTN_ERR_INVALID;
  pages::FreeArgs a{};
  a.window = ll_min(window, 1ll << 40); a.sinks = num_sinks;
  a.table_out = table_out; a.freed = freed; a.count = count;
  return pages::free_pages(c, a, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}

size_t attn_paged_compact_workspace_size(const attn_paged_cache_t* c) {
  if (!pages::cache_ok(c, false, false)) return 0;
  return pages::map_bytes(c) + 3 * align256((size_t)c->num_blocks * 4) + 256;
}

int attn_paged_compact(const attn_paged_cache_t* c, int32_t* table_out, int32_t* num_live, void* workspace,
                       size_t workspace_bytes, void* stream) {
  if (!pages::cache_ok(c, true, true) || !table_out || !num_live) return ATTN_ERR_INVALID;
  if (pages::addr(workspace) % 4) return ATTN_ERR_INVALID;
  if (!workspace || workspace_bytes < attn_paged_compact_workspace_size(c)) return ATTN_ERR_WORKSPACE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  char* ws = reinterpret_cast<char*>(workspace);
  const size_t list = align256((size_t)c->num_blocks * 4);
  pages::CompactArgs a;
  a.table = c->block_table;
  a.entries = (long long)c->num_seqs * c->max_blocks_per_seq;
  a.num_blocks = c->num_blocks;
  a.table_out = table_out; a.num_live = num_live;
  a.live = reinterpret_cast<uint32_t*>(ws);
  a.holes = reinterpret_cast<int32_t*>(ws + pages::map_bytes(c));
  a.movers = reinterpret_cast<int32_t*>(ws + pages::map_bytes(c) + list);
  a.rank = reinterpret_cast<int32_t*>(ws + pages::map_bytes(c) + 2 * list);
  a.moves = reinterpret_cast<int32_t*>(ws + pages::map_bytes(c) + 3 * list);
  const int entry_ctas = (int)ll_min((a.entries + 1023) / 1024, 148);
  int launches = 2;
  if (c->num_blocks <= pages::kClusterPages) {
    static std::atomic<unsigned long long> done{0};
    if (!pages::cluster_smem(pages::compact_cluster_kernel, 1, done)) return ATTN_ERR_CUDA;
    pages::compact_cluster_kernel<<<pages::kCluster, 1024, (c->num_blocks + 31) / 32 * 4, st>>>(a);
  } else {
    if (cudaMemsetAsync(a.live, 0, pages::map_bytes(c), st) != cudaSuccess) return ATTN_ERR_CUDA;
    pages::compact_mark_kernel<<<entry_ctas, 256, 0, st>>>(a);
    pages::compact_list_kernel<<<1, 1024, 0, st>>>(a);
    launches = 3;
  }
  int vec;
  const pages::Pool p = pages::make_pool(c, &vec);
  const int copiers = (int)ll_min(c->num_blocks / 2 + 1, 148 * 8);
#define CALL(V) launch_overlapped(pages::compact_move_kernel<V>, dim3(copiers + entry_ctas), dim3(256), 0, st, p, a, copiers)
  PAGES_BY_VEC(vec, CALL);
#undef CALL
  return launch_status(launches);
}

int attn_paged_accept(const attn_paged_cache_t* c, const void* draft_keys, const void* draft_values,
                      const int64_t k_strides[3], const int64_t v_strides[3], int32_t num_drafts,
                      const int32_t* accepted, int32_t max_accepted, const int32_t* accepted_lengths,
                      int32_t* lengths_out, int32_t* bad, void* stream) {
  if (!pages::cache_ok(c, true, true) || !draft_keys || !draft_values || !k_strides || !v_strides || num_drafts <= 0 ||
      max_accepted < 0 || (max_accepted > 0 && !accepted) || !accepted_lengths || (!lengths_out && !bad))
    return ATTN_ERR_INVALID;
  if (pages::codes(c)) return ATTN_ERR_UNSUPPORTED;      // (their scales: attn_paged_append_tokens)
  if (c->num_seqs > 65535) return ATTN_ERR_UNSUPPORTED;  // (a grid dimension)
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const long long es = dtype_size(c->dtype), row = c->head_dim * es;
  int vec = pages::vec_bytes(row, pages::addr(c->key_pool) | pages::addr(c->value_pool) | pages::addr(draft_keys) |
                                      pages::addr(draft_values));
  for (const int64_t* s : {k_strides, v_strides})
    for (int i = 0; i < 3; ++i)
      while (vec > es && s[i] * es % vec) vec /= 2;
  pages::AcceptArgs a;
  a.table = c->block_table; a.lens = c->seq_lengths; a.accepted = accepted; a.acc_lens = accepted_lengths;
  a.num_seqs = c->num_seqs; a.max_blocks = c->max_blocks_per_seq;
  a.num_blocks = c->num_blocks; a.block_size = c->block_size;
  a.heads = c->num_heads_kv; a.row_vecs = (int)(row / vec);
  a.drafts = num_drafts; a.max_acc = max_accepted;
  a.dk = draft_keys; a.dv = draft_values;
  for (int i = 0; i < 3; ++i) {
    a.ks[i] = k_strides[i] * es / vec;
    a.vs[i] = v_strides[i] * es / vec;
  }
  a.k = c->key_pool; a.v = c->value_pool;
  a.lens_out = lengths_out; a.bad = bad;
  if (bad) {
    pages::accept_check_kernel<<<c->num_seqs, 128, 0, st>>>(a);
    return launch_status();
  }
  const long long per_seq = (long long)max_accepted * a.heads * a.row_vecs;
  if (per_seq > (1ll << 30)) return ATTN_ERR_UNSUPPORTED;
  const unsigned ctas = (unsigned)ll_max((per_seq + 255) / 256, 1);
#define CALL(V) pages::accept_kernel<V><<<dim3(ctas, c->num_seqs), 256, 0, st>>>(a)
  PAGES_BY_VEC(vec, CALL);
#undef CALL
  return launch_status();
}

}  // extern "C"
