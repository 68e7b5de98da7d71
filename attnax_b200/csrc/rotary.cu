// Rotary positions, and tokens that go into a paged cache or come out of it.
//
// A pair (a, b) at position p turns by the angle p w:
//   a' = m (a cos - b sin), b' = m (a sin + b cos);
// the gradient turns by -p w.  Frequencies come as fixed point: w / 2 pi as a
// fraction of 2^64, so p times it modulo 2^64 is the angle's fraction of a
// turn, exact to p 2^-65 turns at any position, and 32 bits of it are enough
// for fp32 sines.  No cos/sin tables are read: the tensors' own bytes are all
// that moves (x once in, once out; 3 flops per element), so HBM bounds the
// large calls and launch latency the small ones.  A thread computes the sines
// of its pairs once and walks over the heads with them.
//
// 8-bit pages: the codes of one page and kv head stand for code * s with
// s = 2^k, the least power of two (2^-100 at least) that brings the largest
// magnitude into the type (448 for e4m3, 127 for int8).  A power of two makes
// the division exact, so a code carries one rounding, and a page whose scale
// grows is restated by an exact quotient (e4m3 codes keep their bits unless
// they become subnormal; int8 codes round once more).
#include <cuda_fp8.h>

#include <climits>
#include <type_traits>

#include "attn_common.cuh"
#include "host_util.h"
#include "sm100.cuh"

namespace attnb200 {
namespace rotary {

struct Spec {
  const unsigned long long* turns;  // [rot / 2], or null: nothing turns
  int rot, interleaved;
  float magnitude, sign;
};

// cos and sin of p w.  The fraction of a turn is cut to the nearest quarter
// turn and a rest of at most pi / 4, where the Taylor series of sine and
// cosine end below 2^-25 after the terms x^9 and x^10.
__device__ __forceinline__ void cos_sin(long long p, unsigned long long turn, float* c, float* s) {
  const unsigned long long f = (unsigned long long)p * turn + 0x80000000ull;
  const int t = (int)(f >> 32);
  const int q = (int)(((unsigned)t + 0x20000000u) >> 30);
  const float x = (float)(t - (int)((unsigned)q << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float z = x * x;
  float sn = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  sn = fmaf(z, sn, 8.3333333e-3f);
  sn = fmaf(z, sn, -1.6666667e-1f);
  sn = fmaf(x * z, sn, x);
  float cs = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  cs = fmaf(z, cs, -1.3888889e-3f);
  cs = fmaf(z, cs, 4.1666667e-2f);
  cs = fmaf(z, cs, -0.5f);
  cs = fmaf(z, cs, 1.f);
  const float a = (q & 1) ? sn : cs, b = (q & 1) ? cs : sn;
  *c = (q == 1 || q == 2) ? -a : a;
  *s = (q & 2) ? -b : b;
}

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T e[N];
};

// One item: NP pairs, in two vectors of NP elements at o1 and o2, or elements behind the turned part.
struct Item {
  int o1, o2;
  bool turned, second;  // second: o2 is inside the head
};

template <int NP>
__device__ __forceinline__ Item item_at(int c, int rot, int dim, bool interleaved) {
  const int pairs = rot / 2 / NP;
  if (c < pairs) return interleaved ? Item{2 * NP * c, 2 * NP * c + NP, true, true} : Item{NP * c, rot / 2 + NP * c, true, true};
  const int o = rot + 2 * NP * (c - pairs);
  return Item{o, o + NP, false, o + NP < dim};
}

__host__ __device__ inline int items_of(int np, int rot, int dim) { return rot / 2 / np + (dim - rot + 2 * np - 1) / (2 * np); }

template <int NP>
__device__ __forceinline__ void item_angles(const Spec& sp, long long pos, int c, float (&cs)[NP], float (&sn)[NP]) {
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    cos_sin(pos, sp.turns[c * NP + j], &cs[j], &sn[j]);
    cs[j] *= sp.magnitude;
    sn[j] *= sp.magnitude * sp.sign;
  }
}

// Values v[0 .. NP) at o1 and v[NP .. 2 NP) at o2, turned.  (A single pair, NP = 1, is (v[0], v[1]) in both layouts.)
template <int NP>
__device__ __forceinline__ void turn(float (&v)[2 * NP], const float (&cs)[NP], const float (&sn)[NP], bool interleaved) {
  if (NP > 1 && interleaved) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const float a = v[2 * j], b = v[2 * j + 1];
      v[2 * j] = a * cs[j] - b * sn[j];
      v[2 * j + 1] = a * sn[j] + b * cs[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const float a = v[j], b = v[NP + j];
      v[j] = a * cs[j] - b * sn[j];
      v[NP + j] = a * sn[j] + b * cs[j];
    }
  }
}

template <typename T, int NP>
__device__ __forceinline__ void load_item(const T* row, const Item& it, float (&v)[2 * NP]) {
  using V = Vec<T, NP>;
  const V a = *reinterpret_cast<const V*>(row + it.o1);
  V b{};
  if (it.second) b = *reinterpret_cast<const V*>(row + it.o2);
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    v[j] = to_f32(a.e[j]);
    v[NP + j] = to_f32(b.e[j]);
  }
}

template <typename T, int NP>
__device__ __forceinline__ void store_item(T* row, const Item& it, const float (&v)[2 * NP]) {
  using V = Vec<T, NP>;
  V a, b;
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    a.e[j] = from_f32<T>(v[j]);
    b.e[j] = from_f32<T>(v[NP + j]);
  }
  *reinterpret_cast<V*>(row + it.o1) = a;
  if (it.second) *reinterpret_cast<V*>(row + it.o2) = b;
}

// A (batch, heads, seq, dim) tensor with unit stride on dim; strides in elements.
struct Rows {
  const void* x;
  void* out;
  long long xs[3], os[3];
  int heads;
};

// ------------------------------------------------------------------ rotary --
struct Args {
  Rows t[2];
  Spec sp;
  const void* positions;
  long long ps[2];
  int positions_64, batch, seq, dim, items, head_group;
};

// Thread = (token, item); it walks over the head_group heads of blockIdx.y
// (of both tensors in a row), kUnroll of them in flight.
template <typename T, int NP>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ Args a) {
  const long long w = blockIdx.x * 256ll + threadIdx.x;
  const long long tok = w / a.items;
  if (tok >= (long long)a.batch * a.seq) return;
  const int c = (int)(w % a.items);
  const int b = (int)(tok / a.seq), s = (int)(tok % a.seq);
  const Item it = item_at<NP>(c, a.sp.rot, a.dim, a.sp.interleaved);
  float cs[NP], sn[NP];
  if (it.turned) {
    long long pos = s;
    if (a.positions) {
      const long long at = b * a.ps[0] + s * a.ps[1];
      pos = a.positions_64 ? reinterpret_cast<const long long*>(a.positions)[at]
                           : reinterpret_cast<const int*>(a.positions)[at];
    }
    item_angles<NP>(a.sp, pos, c, cs, sn);
  }
  const int h1 = min((int)(blockIdx.y + 1) * a.head_group, a.t[0].heads + a.t[1].heads);
#pragma unroll 2
  for (int h = blockIdx.y * a.head_group; h < h1; ++h) {
    const bool second = h >= a.t[0].heads;
    const Rows& r = a.t[second];
    const int hh = second ? h - a.t[0].heads : h;
    float v[2 * NP];
    load_item<T, NP>(reinterpret_cast<const T*>(r.x) + b * r.xs[0] + hh * r.xs[1] + s * r.xs[2], it, v);
    if (it.turned) turn<NP>(v, cs, sn, a.sp.interleaved);
    store_item<T, NP>(reinterpret_cast<T*>(r.out) + b * r.os[0] + hh * r.os[1] + s * r.os[2], it, v);
  }
}

// ------------------------------------------------------------------ append --
struct AppendArgs {
  Rows q, k, v;  // q.heads may be 0; k.out and v.out are the pools
  Spec sp;
  float *ks, *vs;
  const int32_t *table, *lens, *new_lens;
  int32_t *lens_out, *bad;
  int num_seqs, max_blocks, num_blocks, bs, dim, num_new, items, head_group, page_slots, q_ctas;
};

__device__ __forceinline__ int new_tokens(const AppendArgs& a, int s) {
  return a.new_lens ? min(max(a.new_lens[s], 0), a.num_new) : a.num_new;
}

// The page that position `pos` of sequence s is written to, or -1.
__device__ __forceinline__ int write_page(const AppendArgs& a, int s, long long pos) {
  if (pos < 0 || pos / a.bs >= a.max_blocks) return -1;
  const int page = a.table[(long long)s * a.max_blocks + pos / a.bs];
  return page >= 0 && page < a.num_blocks ? page : -1;
}

__device__ __forceinline__ void skip_notice() { atomicCAS(&g_notice, 0, kNoticePageList); }

__device__ __forceinline__ void write_length(const AppendArgs& a, int s) {
  const int n = new_tokens(a, s);
  a.lens_out[s] = a.lens[s] + n;
  if (a.new_lens && n != a.new_lens[s]) skip_notice();
}

__global__ void append_check_kernel(const __grid_constant__ AppendArgs a) {
  const int s = blockIdx.x, n = new_tokens(a, s);
  bool bad = a.new_lens && n != a.new_lens[s];
  for (int i = threadIdx.x; i < n; i += blockDim.x) bad = bad || write_page(a, s, (long long)a.lens[s] + i) < 0;
  if (bad) atomicMin(a.bad, s);
}

// Pools of TO from rows of TI: one rounding, after the turn.  Thread = (token,
// item) as in rotary_kernel, over query heads, key heads and value heads.
template <typename TI, typename TO, int NP>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendArgs a) {
  const long long w = blockIdx.x * 256ll + threadIdx.x;
  const long long tok = w / a.items;
  if (tok >= (long long)a.num_seqs * a.num_new) return;
  const int c = (int)(w % a.items);
  const int s = (int)(tok / a.num_new), i = (int)(tok % a.num_new);
  const bool first = c == 0 && blockIdx.y == 0;
  if (first && i == 0) write_length(a, s);
  const long long pos = (long long)a.lens[s] + i;
  const bool there = i < new_tokens(a, s);
  const int page = there ? write_page(a, s, pos) : -1;
  if (there && page < 0 && first) skip_notice();
  const Item it = item_at<NP>(c, a.sp.rot, a.dim, a.sp.interleaved);
  float cs[NP], sn[NP];
  if (it.turned) item_angles<NP>(a.sp, pos, c, cs, sn);
  const int hq = a.q.heads, hk = a.k.heads;
  const int h1 = min((int)(blockIdx.y + 1) * a.head_group, hq + 2 * hk);
  const long long slot = ((long long)page * a.bs + pos % a.bs) * hk;
#pragma unroll 2
  for (int h = blockIdx.y * a.head_group; h < h1; ++h) {
    float v[2 * NP];
    if (h < hq) {
      load_item<TI, NP>(reinterpret_cast<const TI*>(a.q.x) + s * a.q.xs[0] + h * a.q.xs[1] + i * a.q.xs[2], it, v);
      if (it.turned) turn<NP>(v, cs, sn, a.sp.interleaved);
      store_item<TI, NP>(reinterpret_cast<TI*>(a.q.out) + s * a.q.os[0] + h * a.q.os[1] + i * a.q.os[2], it, v);
    } else if (page >= 0) {
      const bool key = h < hq + hk;
      const Rows& r = key ? a.k : a.v;
      const int hh = key ? h - hq : h - hq - hk;
      load_item<TI, NP>(reinterpret_cast<const TI*>(r.x) + s * r.xs[0] + hh * r.xs[1] + i * r.xs[2], it, v);
      if (key && it.turned) turn<NP>(v, cs, sn, a.sp.interleaved);
      store_item<TO, NP>(reinterpret_cast<TO*>(r.out) + (slot + hh) * a.dim, it, v);
    }
  }
}

// --------------------------------------------------------------- 8-bit codes --
struct E4m3 {
  // 448 = 1.75 * 2^8
  static constexpr int kExp = 8, kTop = 119;  // (a larger scale has codes beyond fp32: the code saturates instead)
  static constexpr uint32_t kMant = 0x600000u;
  static constexpr bool kHasNan = true;
  __device__ static uint8_t code(float x) { return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }
  __device__ static float value(uint8_t c) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3))); }
};
struct Int8 {
  // 127 = 1.984375 * 2^6
  static constexpr int kExp = 6, kTop = 121;
  static constexpr uint32_t kMant = 0x7e0000u;
  static constexpr bool kHasNan = false;
  // (NaN becomes 0: the page's scale is NaN then)
  __device__ static uint8_t code(float x) { return (uint8_t)(int8_t)min(max(__float2int_rn(x), -127), 127); }
  __device__ static float value(uint8_t c) { return (float)(int8_t)c; }
};

// The scale's exponent for the largest finite magnitude `amax`.
template <typename F>
__device__ __forceinline__ int scale_exp(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int k = (int)(u >> 23) - 127 - F::kExp + ((u & 0x7fffffu) > F::kMant);
  return min(max(k, -100), F::kTop);
}
__device__ __forceinline__ float pow2(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }  // |k| <= 126

// Of the rows that go into one page for one kv head: the items' values.
template <typename TI, int NP>
__device__ __forceinline__ void page_item(const AppendArgs& a, const Rows& r, bool key, int s, int h, int i, int c,
                                          long long pos, float (&v)[2 * NP]) {
  const Item it = item_at<NP>(c, a.sp.rot, a.dim, a.sp.interleaved);
  load_item<TI, NP>(reinterpret_cast<const TI*>(r.x) + s * r.xs[0] + h * r.xs[1] + i * r.xs[2], it, v);
  if (key && it.turned) {
    float cs[NP], sn[NP];
    item_angles<NP>(a.sp, pos, c, cs, sn);
    turn<NP>(v, cs, sn, a.sp.interleaved);
  }
}

// CTA = one page of one sequence that gets new tokens, one kv head, keys or
// values; CTAs behind them turn the query.  All tokens of the page are one
// CTA's, so its scale has one writer.
template <typename TI, typename F, int NP>
__global__ void __launch_bounds__(128) append8_kernel(const __grid_constant__ AppendArgs a) {
  if (blockIdx.x < a.q_ctas) {
    const long long w = blockIdx.x * 128ll + threadIdx.x;
    const long long tok = w / a.items;
    const int group = blockIdx.y;  // (gridDim.y groups of head_group heads)
    if (tok >= (long long)a.num_seqs * a.num_new) return;
    const int c = (int)(w % a.items), s = (int)(tok / a.num_new), i = (int)(tok % a.num_new);
    const Item it = item_at<NP>(c, a.sp.rot, a.dim, a.sp.interleaved);
    float cs[NP], sn[NP];
    if (it.turned) item_angles<NP>(a.sp, (long long)a.lens[s] + i, c, cs, sn);
    for (int h = group * a.head_group; h < min((group + 1) * a.head_group, a.q.heads); ++h) {
      float v[2 * NP];
      load_item<TI, NP>(reinterpret_cast<const TI*>(a.q.x) + s * a.q.xs[0] + h * a.q.xs[1] + i * a.q.xs[2], it, v);
      if (it.turned) turn<NP>(v, cs, sn, a.sp.interleaved);
      store_item<TI, NP>(reinterpret_cast<TI*>(a.q.out) + s * a.q.os[0] + h * a.q.os[1] + i * a.q.os[2], it, v);
    }
    return;
  }
  if (blockIdx.y) return;
  const int hk = a.k.heads;
  int x = blockIdx.x - a.q_ctas;
  const int h = x % hk;
  x /= hk;
  const bool key = x & 1;
  x >>= 1;
  const int j = x % a.page_slots, s = x / a.page_slots;
  if (s >= a.num_seqs) return;
  if (j == 0 && h == 0 && key && threadIdx.x == 0) write_length(a, s);
  const int n = new_tokens(a, s);
  const long long len = a.lens[s];
  if (n == 0 || len < 0) {
    if (n && j == 0 && threadIdx.x == 0) skip_notice();
    return;
  }
  const long long p0 = (len / a.bs + j) * a.bs;  // the page's first position
  if (p0 >= len + n) return;
  const int page = write_page(a, s, p0);
  if (page < 0) {
    if (threadIdx.x == 0) skip_notice();
    return;
  }
  const int old = (int)ll_max(len - p0, 0);                    // tokens that were there
  const int count = (int)(ll_min(len + n, p0 + a.bs) - p0) - old;  // new ones, in front of them i0 of the call's
  const int i0 = (int)(p0 + old - len);
  const Rows& r = key ? a.k : a.v;
  const int total = count * a.items;
  float v0[2 * NP];
  float amax = 0.f;
  bool odd = false;
  for (int w = threadIdx.x; w < total; w += 128) {
    float v[2 * NP];
    const int i = i0 + w / a.items;
    page_item<TI, NP>(a, r, key, s, h, i, w % a.items, len + i, v);
#pragma unroll
    for (int e = 0; e < 2 * NP; ++e) {
      const float m = fabsf(v[e]);
      const bool fin = m <= FLT_MAX;
      amax = fin ? fmaxf(amax, m) : amax;
      odd = odd || !fin;
      if (w == threadIdx.x) v0[e] = v[e];
    }
  }
  float* scales = key ? a.ks : a.vs;
  const float s_old = old ? scales[(long long)page * hk + h] : 0.f;  // (read by all before one of them writes it)
  __shared__ float part[4];
  for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = amax;
  odd = __syncthreads_or(odd);
  amax = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  uint8_t* pool = reinterpret_cast<uint8_t*>(r.out);
  const long long row0 = (long long)page * a.bs * hk + h;
  const float need = pow2(scale_exp<F>(amax));
  float s_new = s_old > need ? s_old : need;
  const float inv = 1.f / s_new;
  // int8 has no NaN: a page that was given one has a NaN scale, until it is begun anew
  if (!F::kHasNan && (odd || isnan(s_old))) s_new = NAN;
  for (int w = threadIdx.x; w < total; w += 128) {
    float v[2 * NP];
    const int i = i0 + w / a.items;
    if (w != threadIdx.x) {
      page_item<TI, NP>(a, r, key, s, h, i, w % a.items, len + i, v);
    } else {
#pragma unroll
      for (int e = 0; e < 2 * NP; ++e) v[e] = v0[e];
    }
    const Item it = item_at<NP>(w % a.items, a.sp.rot, a.dim, a.sp.interleaved);
    Vec<uint8_t, NP> c1, c2;
#pragma unroll
    for (int e = 0; e < NP; ++e) {
      // (infinities count as NaN: neither type has them)
      c1.e[e] = F::code(fabsf(v[e]) <= FLT_MAX ? v[e] * inv : NAN);
      c2.e[e] = F::code(fabsf(v[NP + e]) <= FLT_MAX ? v[NP + e] * inv : NAN);
    }
    uint8_t* row = pool + (row0 + (long long)(old + w / a.items) * hk) * a.dim;
    *reinterpret_cast<Vec<uint8_t, NP>*>(row + it.o1) = c1;
    if (it.second) *reinterpret_cast<Vec<uint8_t, NP>*>(row + it.o2) = c2;
  }
  if (threadIdx.x == 0 && !(old && s_new == s_old)) scales[(long long)page * hk + h] = s_new;
  if (old && s_new > s_old) {  // (never with a NaN)
    const float ratio = s_old / s_new;
    for (int w = threadIdx.x; w < old * a.dim; w += 128) {
      uint8_t* at = pool + (row0 + (long long)(w / a.dim) * hk) * a.dim + w % a.dim;
      *at = F::code(F::value(*at) * ratio);
    }
  }
}

// ------------------------------------------------------------------ gather --
struct GatherArgs {
  const void *k, *v;
  const float *ks, *vs;
  void *ko, *vo;
  const int32_t *table, *lens, *starts;
  int num_seqs, max_blocks, num_blocks, bs, hk, dim, count, vecs;
};

template <typename F, typename TO>
__device__ __forceinline__ TO gather_value(const void* pool, long long at, float scale) {
  if constexpr (std::is_same<F, E4m3>::value || std::is_same<F, Int8>::value)
    return from_f32<TO>(F::value(reinterpret_cast<const uint8_t*>(pool)[at]) * scale);
  else
    return from_f32<TO>(to_f32(reinterpret_cast<const F*>(pool)[at]));
}

// Thread = NV elements of one token's kv head, of keys (blockIdx.y 0) or
// values; positions outside the sequence give zeros.
template <typename F, typename TO, int NV>
__global__ void __launch_bounds__(256) gather_tokens_kernel(const __grid_constant__ GatherArgs a) {
  const long long w = blockIdx.x * 256ll + threadIdx.x;
  const long long per_tok = (long long)a.hk * a.vecs;
  const long long t = w / per_tok;
  if (t >= (long long)a.num_seqs * a.count) return;
  const int x = (int)(w % per_tok), h = x / a.vecs, e = x % a.vecs * NV;
  const int s = (int)(t / a.count);
  const long long pos = (a.starts ? a.starts[s] : 0ll) + t % a.count;
  Vec<TO, NV> o;
#pragma unroll
  for (int j = 0; j < NV; ++j) o.e[j] = from_f32<TO>(0.f);
  if (pos >= 0 && pos < a.lens[s]) {
    if (pos / a.bs >= a.max_blocks) {
      atomicCAS(&g_notice, 0, kNoticeTableOverrun);
    } else {
      const long long page = paged_phys_page(a.table[(long long)s * a.max_blocks + pos / a.bs], a.num_blocks);
      const long long at = ((page * a.bs + pos % a.bs) * a.hk + h) * a.dim + e;
      const void* pool = blockIdx.y ? a.v : a.k;
      float scale = 1.f;
      constexpr bool bits8 = std::is_same<F, E4m3>::value || std::is_same<F, Int8>::value;
      if (bits8) scale = (blockIdx.y ? a.vs : a.ks)[page * a.hk + h];
      using S = typename std::conditional<bits8, uint8_t, F>::type;
      const Vec<S, NV> in = *reinterpret_cast<const Vec<S, NV>*>(reinterpret_cast<const S*>(pool) + at);
#pragma unroll
      for (int j = 0; j < NV; ++j) o.e[j] = gather_value<F, TO>(&in, j, scale);
    }
  }
  TO* out = reinterpret_cast<TO*>(blockIdx.y ? a.vo : a.ko);
  *reinterpret_cast<Vec<TO, NV>*>(out + (t * a.hk + h) * a.dim + e) = o;
}

// -------------------------------------------------------------------- host --
static uintptr_t addr(const void* p) { return reinterpret_cast<uintptr_t>(p); }
static bool dtype_ok(int t) { return t == ATTN_F32 || t == ATTN_BF16 || t == ATTN_F16; }

// Whether vectors of `bytes` fit the address and the strides that are stepped (elements of `es` bytes).
static bool fits(const void* p, const long long* strides, long long es, int bytes) {
  if (addr(p) % bytes) return false;
  for (int i = 0; i < 3; ++i)
    if (strides[i] * es % bytes) return false;
  return true;
}

static bool spec_ok(const attn_rotary_spec_t& r, int dim) {
  return !r.turns || (r.rotary_dim > 0 && r.rotary_dim % 2 == 0 && r.rotary_dim <= dim);
}

static Spec make_spec(const attn_rotary_spec_t& r, float sign) {
  return Spec{reinterpret_cast<const unsigned long long*>(r.turns), r.turns ? r.rotary_dim : 0, r.interleaved != 0,
              r.magnitude, sign};
}

static Rows make_rows(const void* x, const int64_t* xs, void* out, const int64_t* os, int heads) {
  Rows r{};
  r.x = x; r.out = out; r.heads = heads;
  for (int i = 0; i < 3; ++i) {
    r.xs[i] = xs ? xs[i] : 0;
    r.os[i] = os ? os[i] : 0;
  }
  return r;
}

// Heads per thread: as many as leave about two waves of threads, so that the sines are shared but no SM is idle.
static int head_group(long long threads, int heads) {
  const long long want = 148ll * 2048 * 2;
  long long groups = ll_min(heads, ll_max(1, (want + threads - 1) / threads));
  groups = ll_min(groups, 65535);
  return (int)((heads + groups - 1) / groups);
}

}  // namespace rotary

bool rotary_take_status(int* status, int* notice) { return take_status_words(status, notice); }

}  // namespace attnb200

using namespace attnb200;

// Runs CALL(NP) with NP the widest of 16 bytes, 8 bytes and one element that `ok` allows.
#define BY_WIDTH(es, ok, CALL)      \
  do {                              \
    if (es == 4) {                  \
      if (ok(4)) CALL(4);           \
      else if (ok(2)) CALL(2);      \
      else CALL(1);                 \
    } else {                        \
      if (ok(8)) CALL(8);           \
      else if (ok(4)) CALL(4);      \
      else CALL(1);                 \
    }                               \
  } while (0)

extern "C" {

int attn_rotary(const attn_rotary_params_t* p, void* stream) {
  using namespace rotary;
  if (!p || !dtype_ok(p->dtype) || p->batch < 0 || p->seq < 0 || p->head_dim <= 0 || p->heads_q < 0 || p->heads_k < 0 ||
      !p->rotary.turns || !spec_ok(p->rotary, p->head_dim))
    return ATTN_ERR_INVALID;
  const long long tokens = (long long)p->batch * p->seq;
  const int heads = p->heads_q + p->heads_k;
  if (tokens == 0 || heads == 0) return ATTN_OK;
  if ((p->heads_q && (!p->q || !p->q_out)) || (p->heads_k && (!p->k || !p->k_out))) return ATTN_ERR_INVALID;
  Args a{};
  a.t[0] = make_rows(p->q, p->q_strides, p->q_out, p->q_out_strides, p->heads_q);
  a.t[1] = make_rows(p->k, p->k_strides, p->k_out, p->k_out_strides, p->heads_k);
  a.sp = make_spec(p->rotary, p->inverse ? -1.f : 1.f);
  a.positions = p->positions;
  a.positions_64 = p->positions_64;
  a.ps[0] = p->position_strides[0]; a.ps[1] = p->position_strides[1];
  a.batch = p->batch; a.seq = p->seq; a.dim = p->head_dim;
  const int es = (int)dtype_size(p->dtype);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto ok = [&](int np) {
    if (a.sp.rot / 2 % np || a.dim % np) return false;
    for (const Rows& r : a.t)
      if (r.heads && !(fits(r.x, r.xs, es, np * es) && fits(r.out, r.os, es, np * es))) return false;
    return true;
  };
#define LAUNCH(T, NP)                                                                  \
  do {                                                                                 \
    a.items = items_of(NP, a.sp.rot, a.dim);                                           \
    const long long threads = tokens * a.items;                                        \
    if ((threads + 255) / 256 > INT_MAX) return ATTN_ERR_UNSUPPORTED;                  \
    a.head_group = head_group(threads, heads);                                         \
    const dim3 grid((unsigned)((threads + 255) / 256), (heads + a.head_group - 1) / a.head_group); \
    rotary_kernel<T, NP><<<grid, 256, 0, st>>>(a);                                     \
  } while (0)
#define CALL(NP)                                              \
  do {                                                        \
    if (p->dtype == ATTN_F32) LAUNCH(float, (NP > 4 ? 4 : NP)); \
    else if (p->dtype == ATTN_BF16) LAUNCH(__nv_bfloat16, NP); \
    else LAUNCH(__half, NP);                                  \
  } while (0)
  BY_WIDTH(es, ok, CALL);
#undef CALL
#undef LAUNCH
  return launch_status();
}

int attn_paged_append_tokens(const attn_paged_append_params_t* p, void* stream) {
  using namespace rotary;
  if (!p || !dtype_ok(p->dtype) || p->num_blocks <= 0 || p->block_size <= 0 || p->num_heads_kv <= 0 ||
      p->head_dim <= 0 || p->num_seqs <= 0 || p->max_blocks_per_seq <= 0 || p->num_new <= 0 || !p->key_pool ||
      !p->value_pool || !p->block_table || !p->seq_lengths || !p->keys || !p->values || p->num_heads_q < 0 ||
      (p->num_heads_q && (!p->q || !p->q_out)) || (!p->lengths_out && !p->bad) || !spec_ok(p->rotary, p->head_dim))
    return ATTN_ERR_INVALID;
  const bool bits8 = p->pool_format == ATTN_POOL_E4M3 || p->pool_format == ATTN_POOL_INT8;
  if (!bits8 && !dtype_ok(p->pool_format)) return ATTN_ERR_INVALID;
  if (bits8 && (!p->key_scales || !p->value_scales)) return ATTN_ERR_INVALID;
  AppendArgs a{};
  a.q = make_rows(p->q, p->q_strides, p->q_out, p->q_out_strides, p->num_heads_q);
  a.k = make_rows(p->keys, p->k_strides, p->key_pool, nullptr, p->num_heads_kv);
  a.v = make_rows(p->values, p->v_strides, p->value_pool, nullptr, p->num_heads_kv);
  a.sp = make_spec(p->rotary, 1.f);
  a.ks = p->key_scales; a.vs = p->value_scales;
  a.table = p->block_table; a.lens = p->seq_lengths; a.new_lens = p->new_lengths;
  a.lens_out = p->lengths_out; a.bad = p->bad;
  a.num_seqs = p->num_seqs; a.max_blocks = p->max_blocks_per_seq; a.num_blocks = p->num_blocks;
  a.bs = p->block_size; a.dim = p->head_dim; a.num_new = p->num_new;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p->bad) {
    append_check_kernel<<<a.num_seqs, 128, 0, st>>>(a);
    return launch_status();
  }
  const int es = (int)dtype_size(p->dtype);
  const int po = bits8 ? 1 : (int)dtype_size((attn_dtype_t)p->pool_format);
  auto ok = [&](int np) {
    if (a.sp.rot / 2 % np || a.dim % np || (addr(a.k.out) | addr(a.v.out)) % (np * po)) return false;
    for (const Rows* r : {&a.k, &a.v})
      if (!fits(r->x, r->xs, es, np * es)) return false;
    return !a.q.heads || (fits(a.q.x, a.q.xs, es, np * es) && fits(a.q.out, a.q.os, es, np * es));
  };
  const long long tokens = (long long)a.num_seqs * a.num_new;
#define WIDE(TI, TO, NP)                                                               \
  do {                                                                                 \
    a.items = items_of(NP, a.sp.rot, a.dim);                                           \
    const long long threads = tokens * a.items;                                        \
    const int heads = a.q.heads + 2 * a.k.heads;                                       \
    if ((threads + 255) / 256 > INT_MAX) return ATTN_ERR_UNSUPPORTED;                  \
    a.head_group = head_group(threads, heads);                                         \
    const dim3 grid((unsigned)((threads + 255) / 256), (heads + a.head_group - 1) / a.head_group); \
    append_kernel<TI, TO, NP><<<grid, 256, 0, st>>>(a);                                \
  } while (0)
#define BITS8(TI, F, NP)                                                               \
  do {                                                                                 \
    a.items = items_of(NP, a.sp.rot, a.dim);                                           \
    a.page_slots = (int)(((long long)a.num_new + a.bs - 1) / a.bs) + 1;                \
    const long long pages = (long long)a.num_seqs * a.page_slots * 2 * a.k.heads;      \
    const long long qc = a.q.heads ? (tokens * a.items + 127) / 128 : 0;               \
    if (pages + qc > INT_MAX) return ATTN_ERR_UNSUPPORTED;                             \
    a.q_ctas = (int)qc;                                                                \
    a.head_group = a.q.heads ? head_group(tokens * a.items, a.q.heads) : 1;            \
    const dim3 grid((unsigned)(pages + qc), a.q.heads ? (a.q.heads + a.head_group - 1) / a.head_group : 1); \
    append8_kernel<TI, F, NP><<<grid, 128, 0, st>>>(a);                                \
  } while (0)
#define POOL(TI, NP)                                                    \
  do {                                                                  \
    switch (p->pool_format) {                                           \
      case ATTN_F32: WIDE(TI, float, NP); break;                        \
      case ATTN_BF16: WIDE(TI, __nv_bfloat16, NP); break;               \
      case ATTN_F16: WIDE(TI, __half, NP); break;                       \
      case ATTN_POOL_E4M3: BITS8(TI, E4m3, NP); break;                  \
      default: BITS8(TI, Int8, NP);                                     \
    }                                                                   \
  } while (0)
#define CALL(NP)                                             \
  do {                                                       \
    if (p->dtype == ATTN_F32) POOL(float, (NP > 4 ? 4 : NP)); \
    else if (p->dtype == ATTN_BF16) POOL(__nv_bfloat16, NP); \
    else POOL(__half, NP);                                   \
  } while (0)
  BY_WIDTH(es, ok, CALL);
#undef CALL
#undef POOL
#undef BITS8
#undef WIDE
  return launch_status();
}

int attn_paged_gather_tokens(const attn_paged_gather_params_t* p, void* stream) {
  using namespace rotary;
  if (!p || !dtype_ok(p->dtype) || p->num_blocks <= 0 || p->block_size <= 0 || p->num_heads_kv <= 0 ||
      p->head_dim <= 0 || p->num_seqs < 0 || p->count < 0)
    return ATTN_ERR_INVALID;
  if (p->num_seqs == 0 || p->count == 0) return ATTN_OK;
  const bool bits8 = p->pool_format == ATTN_POOL_E4M3 || p->pool_format == ATTN_POOL_INT8;
  if (!bits8 && !dtype_ok(p->pool_format)) return ATTN_ERR_INVALID;
  if (!p->key_pool || !p->value_pool || !p->block_table || !p->seq_lengths || !p->keys_out || !p->values_out ||
      p->max_blocks_per_seq <= 0 || (bits8 && (!p->key_scales || !p->value_scales)))
    return ATTN_ERR_INVALID;
  GatherArgs a{p->key_pool, p->value_pool, p->key_scales, p->value_scales, p->keys_out, p->values_out, p->block_table,
               p->seq_lengths, p->starts, p->num_seqs, p->max_blocks_per_seq, p->num_blocks, p->block_size,
               p->num_heads_kv, p->head_dim, p->count, 0};
  const int pi = bits8 ? 1 : (int)dtype_size((attn_dtype_t)p->pool_format), po = (int)dtype_size(p->dtype);
  const uintptr_t in = addr(a.k) | addr(a.v), out = addr(a.ko) | addr(a.vo);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool wide = a.dim % 4 == 0 && in % (4 * pi) == 0 && out % (4 * po) == 0;
  const bool wider = bits8 && po == 2 && a.dim % 8 == 0 && in % 8 == 0 && out % 16 == 0;
#define RUN(F, TO, NV)                                                                 \
  do {                                                                                 \
    a.vecs = a.dim / NV;                                                               \
    const long long n = ((long long)a.num_seqs * a.count * a.hk * a.vecs + 255) / 256; \
    if (n > INT_MAX) return ATTN_ERR_UNSUPPORTED;                                      \
    gather_tokens_kernel<F, TO, NV><<<dim3((unsigned)n, 2), 256, 0, st>>>(a);          \
  } while (0)
#define TO_(F, NV)                                             \
  do {                                                         \
    if (p->dtype == ATTN_F32) RUN(F, float, NV);               \
    else if (p->dtype == ATTN_BF16) RUN(F, __nv_bfloat16, NV); \
    else RUN(F, __half, NV);                                   \
  } while (0)
#define W(F)            \
  do {                  \
    if (wide) TO_(F, 4); \
    else TO_(F, 1);     \
  } while (0)
#define W8(F)                                                    \
  do {                                                           \
    if (wider && p->dtype == ATTN_BF16) RUN(F, __nv_bfloat16, 8); \
    else if (wider) RUN(F, __half, 8);                           \
    else W(F);                                                   \
  } while (0)
  switch (p->pool_format) {
    case ATTN_F32: W(float); break;
    case ATTN_BF16: W(__nv_bfloat16); break;
    case ATTN_F16: W(__half); break;
    case ATTN_POOL_E4M3: W8(E4m3); break;
    default: W8(Int8);
  }
#undef W8
#undef W
#undef TO_
#undef RUN
  return launch_status();
}

}  // extern "C"
