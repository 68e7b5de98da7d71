// Rotary positions, and tokens that go into a paged cache or come out of it.
//
// A pair (a, b) at position p turns by the angle p w:
//   a' = m (a cos - b sin), b' = m (a sin + b cos);
// the gradient turns by -p w.  Frequencies come as fixed point: w / 2 pi as a
// fraction of 2^64, so p times it modulo 2^64 is the angle's fraction of a
// turn, exact to p 2^-64 turns at any position, and 32 bits of it are enough
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
  const unsigned t = (unsigned)(f >> 32), q = (t + 0x20000000u) >> 30;
  const float x = (float)(int)(t - (q << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
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

// Vectors are moved as machine words: as structs, the compiler split those that it keeps for several heads into
// elements (training shape, one direction: 280 us instead of 115).
template <int BYTES> struct Word;
template <> struct Word<1> { using T = uint8_t; };
template <> struct Word<2> { using T = uint16_t; };
template <> struct Word<4> { using T = uint32_t; };
template <> struct Word<8> { using T = uint2; };
template <> struct Word<16> { using T = uint4; };
template <typename T, int N>
using Bits = typename Word<sizeof(T) * N>::T;

template <typename T, int N>
__device__ __forceinline__ Vec<T, N> unpack(const Bits<T, N>& w) {
  Vec<T, N> v;
  static_assert(sizeof(v) == sizeof(w), "");
  memcpy(&v, &w, sizeof(v));
  return v;
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* at, const Vec<T, N>& v) {
  constexpr int M = sizeof(T) * N > 16 ? 16 / sizeof(T) : N;
#pragma unroll
  for (int i = 0; i < N / M; ++i) {
    Bits<T, M> w;
    memcpy(&w, v.e + i * M, sizeof(w));
    reinterpret_cast<Bits<T, M>*>(at)[i] = w;
  }
}

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

// An item as it lies in memory.
template <typename T, int NP>
struct Raw {
  Bits<T, NP> a, b;
};
template <typename T, int NP>
__device__ __forceinline__ Raw<T, NP> load_raw(const T* row, const Item& it) {
  Raw<T, NP> r{};
  r.a = *reinterpret_cast<const Bits<T, NP>*>(row + it.o1);
  if (it.second) r.b = *reinterpret_cast<const Bits<T, NP>*>(row + it.o2);
  return r;
}
template <typename T, int NP>
__device__ __forceinline__ void widen(const Raw<T, NP>& r, float (&v)[2 * NP]) {
  const Vec<T, NP> a = unpack<T, NP>(r.a), b = unpack<T, NP>(r.b);
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    v[j] = to_f32(a.e[j]);
    v[NP + j] = to_f32(b.e[j]);
  }
}

template <typename T, int NP>
__device__ __forceinline__ void store_item(T* row, const Item& it, const float (&v)[2 * NP]) {
  Vec<T, NP> a, b;
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    a.e[j] = from_f32<T>(v[j]);
    b.e[j] = from_f32<T>(v[NP + j]);
  }
  store_vec<T, NP>(row + it.o1, a);
  if (it.second) store_vec<T, NP>(row + it.o2, b);
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
  int positions_64, seq, dim, items, head_group, head_lanes, cta_tokens;
  int tokens;
};

// Heads whose loads a thread has in flight together.  (The output may alias the input, so the compiler keeps loads
// behind the stores in front of them: they are issued by hand.)
constexpr int kHeads = 2;

// CTA = cta_tokens tokens and the head_group heads of blockIdx.y, of both tensors in a row; thread = (token, one of
// head_lanes heads in turn, item).  Four head lanes make a warp's accesses neighbours in memory where a token's heads
// lie side by side, one where a head's tokens do.
template <typename T, int NP>
__global__ void __launch_bounds__(256, 3) rotary_kernel(const __grid_constant__ Args a) {
  const int in_cta = threadIdx.x / a.items / a.head_lanes, sub = threadIdx.x / a.items % a.head_lanes;
  const int tok = blockIdx.x * a.cta_tokens + in_cta;
  if (in_cta >= a.cta_tokens || tok >= a.tokens) return;
  const int b = tok / a.seq, s = tok % a.seq;
  long long pos = s;
  if (a.positions) {
    const long long at = b * a.ps[0] + s * a.ps[1];
    pos = a.positions_64 ? reinterpret_cast<const long long*>(a.positions)[at]
                         : reinterpret_cast<const int*>(a.positions)[at];
  }
  const int hq = a.t[0].heads, hl = a.head_lanes;
  const int h0 = blockIdx.y * a.head_group, h1 = min(h0 + a.head_group, hq + a.t[1].heads);
  const T* x0 = reinterpret_cast<const T*>(a.t[0].x) + b * a.t[0].xs[0] + s * a.t[0].xs[2];
  const T* x1 = reinterpret_cast<const T*>(a.t[1].x) + b * a.t[1].xs[0] + s * a.t[1].xs[2];
  T* y0 = reinterpret_cast<T*>(a.t[0].out) + b * a.t[0].os[0] + s * a.t[0].os[2];
  T* y1 = reinterpret_cast<T*>(a.t[1].out) + b * a.t[1].os[0] + s * a.t[1].os[2];
  for (int c = threadIdx.x % a.items; c < a.items; c += 256) {  // (more than 256 items: one token per CTA)
    const Item it = item_at<NP>(c, a.sp.rot, a.dim, a.sp.interleaved);
    float cs[NP], sn[NP];
    if (it.turned) item_angles<NP>(a.sp, pos, c, cs, sn);
    for (int h = h0 + sub; h < h1; h += kHeads * hl) {
      Raw<T, NP> raw[kHeads];
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        const int x = h + u * hl;
        if (x < h1) raw[u] = load_raw<T, NP>(x < hq ? x0 + x * a.t[0].xs[1] : x1 + (x - hq) * a.t[1].xs[1], it);
      }
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        const int x = h + u * hl;
        if (x >= h1) break;
        float v[2 * NP];
        widen<T, NP>(raw[u], v);
        if (it.turned) turn<NP>(v, cs, sn, a.sp.interleaved);
        store_item<T, NP>(x < hq ? y0 + x * a.t[0].os[1] : y1 + (x - hq) * a.t[1].os[1], it, v);
      }
    }
  }
}

// ------------------------------------------------------------------ append --
struct AppendArgs {
  Rows q, k, v;  // q.heads may be 0; k.out and v.out are the pools
  Spec sp;
  float *ks, *vs;
  const int32_t *table, *lens, *new_lens;
  int32_t *lens_out, *bad;
  int num_seqs, max_blocks, num_blocks, bs, dim, num_new, items, head_group, head_lanes, cta_tokens, page_slots, page_heads, page_ctas, q_ctas, angles;
};

__device__ __forceinline__ int new_tokens(const AppendArgs& a, int s) {
  return a.new_lens ? min(max(a.new_lens[s], 0), a.num_new) : a.num_new;
}

// The page that position `pos` of sequence s is written to, or -1 (a sequence whose length is negative has none).
__device__ __forceinline__ int write_page(const AppendArgs& a, int s, long long pos) {
  if (a.lens[s] < 0 || pos / a.bs >= a.max_blocks) return -1;
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

// Pools of TO from rows of TI: one rounding, after the turn.  CTAs and threads as in rotary_kernel, over the query
// heads, the key heads and the value heads of every token.
template <typename TI, typename TO, int NP>
__global__ void __launch_bounds__(256, 3) append_kernel(const __grid_constant__ AppendArgs a) {
  const int in_cta = threadIdx.x / a.items / a.head_lanes, sub = threadIdx.x / a.items % a.head_lanes;
  const int tok = blockIdx.x * a.cta_tokens + in_cta;
  if (in_cta >= a.cta_tokens || tok >= a.num_seqs * a.num_new) return;
  const int s = tok / a.num_new, i = tok % a.num_new;
  const bool first = threadIdx.x % a.items == 0 && sub == 0 && blockIdx.y == 0;
  if (first && i == 0) write_length(a, s);
  const long long pos = (long long)a.lens[s] + i;
  const bool there = i < new_tokens(a, s);
  const int page = there ? write_page(a, s, pos) : -1;
  if (there && page < 0 && first) skip_notice();
  const int hq = a.q.heads, hk = a.k.heads, hl = a.head_lanes, h0 = blockIdx.y * a.head_group;
  const int h1 = min(h0 + a.head_group, page < 0 ? hq : hq + 2 * hk);
  const TI* xq = reinterpret_cast<const TI*>(a.q.x) + s * a.q.xs[0] + i * a.q.xs[2];
  const TI* xk = reinterpret_cast<const TI*>(a.k.x) + s * a.k.xs[0] + i * a.k.xs[2];
  const TI* xv = reinterpret_cast<const TI*>(a.v.x) + s * a.v.xs[0] + i * a.v.xs[2];
  TI* yq = reinterpret_cast<TI*>(a.q.out) + s * a.q.os[0] + i * a.q.os[2];
  const long long slot = ((long long)page * a.bs + pos % a.bs) * hk * a.dim;
  for (int c = threadIdx.x % a.items; c < a.items; c += 256) {
    const Item it = item_at<NP>(c, a.sp.rot, a.dim, a.sp.interleaved);
    float cs[NP], sn[NP];
    if (it.turned && h0 < hq + hk) item_angles<NP>(a.sp, pos, c, cs, sn);
    for (int h = h0 + sub; h < h1; h += kHeads * hl) {
      Raw<TI, NP> raw[kHeads];
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        const int x = h + u * hl;
        if (x < h1)
          raw[u] = load_raw<TI, NP>(x < hq        ? xq + x * a.q.xs[1]
                                    : x < hq + hk ? xk + (x - hq) * a.k.xs[1]
                                                  : xv + (x - hq - hk) * a.v.xs[1],
                                    it);
      }
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        const int x = h + u * hl;
        if (x >= h1) break;
        float v[2 * NP];
        widen<TI, NP>(raw[u], v);
        if (it.turned && x < hq + hk) turn<NP>(v, cs, sn, a.sp.interleaved);
        if (x < hq) store_item<TI, NP>(yq + x * a.q.os[1], it, v);
        else if (x < hq + hk) store_item<TO, NP>(reinterpret_cast<TO*>(a.k.out) + slot + (x - hq) * a.dim, it, v);
        else store_item<TO, NP>(reinterpret_cast<TO*>(a.v.out) + slot + (x - hq - hk) * a.dim, it, v);
      }
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
  // four codes of values in range
  __device__ static uint32_t code4(float a, float b, float c, float d) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) |
           (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16;
  }
};
struct Int8 {
  // 127 = 1.984375 * 2^6
  static constexpr int kExp = 6, kTop = 121;
  static constexpr uint32_t kMant = 0x7e0000u;
  static constexpr bool kHasNan = false;
  // (NaN becomes 0: the page's scale is NaN then)
  __device__ static uint8_t code(float x) { return (uint8_t)(int8_t)min(max(__float2int_rn(x), -127), 127); }
  __device__ static float value(uint8_t c) { return (float)(int8_t)c; }
  // 1.5 * 2^23 + x holds x rounded to even in its low bits (the conversion instruction runs at a quarter of the rate)
  __device__ static uint32_t code4(float a, float b, float c, float d) {
    constexpr float kRound = 12582912.f;
    const uint32_t ab = __byte_perm(__float_as_uint(a + kRound), __float_as_uint(b + kRound), 0x0040);
    const uint32_t cd = __byte_perm(__float_as_uint(c + kRound), __float_as_uint(d + kRound), 0x0040);
    return __byte_perm(ab, cd, 0x5410);
  }
};
// Codes of v[0 .. N) * inv; `careful`: some may be out of range or not finite (infinities count as NaN, which neither
// type tells apart).
template <typename F, int N>
__device__ __forceinline__ Bits<uint8_t, N> codes_of(const float* v, float inv, bool careful) {
  uint32_t w[(N + 3) / 4];
  if (careful) {
#pragma unroll
    for (int i = 0; i < (N + 3) / 4; ++i) {
      w[i] = 0;
#pragma unroll
      for (int e = 0; e < 4 && 4 * i + e < N; ++e)
        w[i] |= (uint32_t)F::code(fabsf(v[4 * i + e]) <= FLT_MAX ? v[4 * i + e] * inv : NAN) << (8 * e);
    }
  } else {
#pragma unroll
    for (int i = 0; i < (N + 3) / 4; ++i) {
      auto at = [&](int e) { return 4 * i + e < N ? v[4 * i + e] * inv : 0.f; };
      w[i] = F::code4(at(0), at(1), at(2), at(3));
    }
  }
  Bits<uint8_t, N> out;
  memcpy(&out, w, sizeof(out));
  return out;
}

// The scale's exponent for the largest finite magnitude `amax`.
template <typename F>
__device__ __forceinline__ int scale_exp(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int k = (int)(u >> 23) - 127 - F::kExp + ((u & 0x7fffffu) > F::kMant);
  return min(max(k, -100), F::kTop);
}
__device__ __forceinline__ float pow2(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }  // |k| <= 126

// The query's CTAs of append8_kernel: cta_tokens tokens and head_group heads, threads as in rotary_kernel.
template <typename T, int NP>
__device__ __forceinline__ void turn_query(const AppendArgs& a, int cta) {
  const int hl = a.head_lanes;
  const int in_cta = threadIdx.x / a.items / hl, sub = threadIdx.x / a.items % hl;
  const int tok = cta % a.q_ctas * a.cta_tokens + in_cta, h0 = cta / a.q_ctas * a.head_group;
  if (in_cta >= a.cta_tokens || tok >= a.num_seqs * a.num_new) return;
  const int s = tok / a.num_new, i = tok % a.num_new, h1 = min(h0 + a.head_group, a.q.heads);
  const T* x = reinterpret_cast<const T*>(a.q.x) + s * a.q.xs[0] + i * a.q.xs[2];
  T* y = reinterpret_cast<T*>(a.q.out) + s * a.q.os[0] + i * a.q.os[2];
  for (int c = threadIdx.x % a.items; c < a.items; c += blockDim.x) {
    const Item it = item_at<NP>(c, a.sp.rot, a.dim, a.sp.interleaved);
    float cs[NP], sn[NP];
    if (it.turned) item_angles<NP>(a.sp, (long long)a.lens[s] + i, c, cs, sn);
    for (int h = h0 + sub; h < h1; h += kHeads * hl) {
      Raw<T, NP> raw[kHeads];
#pragma unroll
      for (int u = 0; u < kHeads; ++u)
        if (h + u * hl < h1) raw[u] = load_raw<T, NP>(x + (h + u * hl) * a.q.xs[1], it);
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        if (h + u * hl >= h1) break;
        float v[2 * NP];
        widen<T, NP>(raw[u], v);
        if (it.turned) turn<NP>(v, cs, sn, a.sp.interleaved);
        store_item<T, NP>(y + (h + u * hl) * a.q.os[1], it, v);
      }
    }
  }
}

constexpr int kPageThreads = 256;
constexpr int kAngleBytes = 40960;  // of shared memory, at most

// page_ctas CTAs: one page of one sequence that gets new tokens, keys or values, and page_heads kv heads one
// after another.  All tokens of a page and head are one CTA's, so a scale has one writer.  The sines of the page's
// tokens are kept in shared memory for all of its heads (`angles` items of them, 0: formed again where they are
// needed).  The others turn the query and lie evenly among them: pages wait for instructions, the query for HBM
// (8 prompts of 4096, 32 heads over 8, e4m3: 181 us, 193 with the query in a launch in front; 16 of 128: 27 against
// 31; four CTAs per SM at 64 registers: 209.  At 80 registers, 16-bit rows in 16-byte vectors spill 144 bytes of stores
// and 80 of loads.)  A thread keeps its first item between the pass for the largest
// magnitude and the one for the codes; a larger page's others are read twice.
template <typename TI, typename F, int NP>
__global__ void __launch_bounds__(kPageThreads, 3) append8_kernel(const __grid_constant__ AppendArgs a) {
  const int query_ctas = gridDim.x - a.page_ctas, before = (int)((long long)blockIdx.x * query_ctas / gridDim.x);
  if ((long long)(blockIdx.x + 1) * query_ctas / gridDim.x > before) {
    turn_query<TI, NP>(a, before);
    return;
  }
  extern __shared__ float2 table[];  // [pair of the item][item]
  const int hk = a.k.heads, tid = threadIdx.x, threads = blockDim.x, lane = tid % 32;
  const int groups = (hk + a.page_heads - 1) / a.page_heads;
  int x = blockIdx.x - before;
  const int h0 = x % groups * a.page_heads, h1 = min(h0 + a.page_heads, hk);
  x /= groups;
  const bool key = x & 1;
  x >>= 1;
  const int j = x % a.page_slots, s = x / a.page_slots;
  const long long len = a.lens[s];
  const int n = new_tokens(a, s);
  if (j == 0 && h0 == 0 && key && tid == 0) write_length(a, s);
  if (n == 0 || len < 0) {
    if (n && j == 0 && tid == 0) skip_notice();
    return;
  }
  const long long p0 = (len / a.bs + j) * a.bs;  // the page's first position
  if (p0 >= len + n) return;
  const int page = write_page(a, s, p0);
  if (page < 0) {
    if (tid == 0) skip_notice();
    return;
  }
  const int old = (int)ll_max(len - p0, 0);                        // tokens that were there
  const int count = (int)(ll_min(len + n, p0 + a.bs) - p0) - old;  // new ones, in front of them i0 of the call's
  const int i0 = (int)(p0 + old - len);
  const Rows& r = key ? a.k : a.v;
  float* const scales = (key ? a.ks : a.vs) + (long long)page * hk;
  const int pool_row = hk * a.dim;
  uint8_t* const pool = reinterpret_cast<uint8_t*>(r.out) + (long long)page * a.bs * pool_row;
  const TI* const rows = reinterpret_cast<const TI*>(r.x) + s * r.xs[0] + i0 * r.xs[2];
  // Thread (i, c) has item c of the tokens i, i + step, ..
  const int c = tid % a.items, step = threads / a.items, i = tid / a.items < step ? tid / a.items : count;
  const Item it = item_at<NP>(c, a.sp.rot, a.dim, a.sp.interleaved);
  const bool turns = key && it.turned;
  if (key && a.angles) {
    if (turns)
      for (int w = i; w < count; w += step) {
        float cs[NP], sn[NP];
        item_angles<NP>(a.sp, len + i0 + w, c, cs, sn);
#pragma unroll
        for (int e = 0; e < NP; ++e) table[e * a.angles + w * a.items + c] = make_float2(cs[e], sn[e]);
      }
    __syncthreads();
  }
  auto load = [&](int h, int w) { return load_raw<TI, NP>(rows + h * r.xs[1] + w * r.xs[2], it); };
  auto values = [&](const Raw<TI, NP>& raw, int w, float (&v)[2 * NP]) {
    widen<TI, NP>(raw, v);
    if (!turns) return;
    float cs[NP], sn[NP];
    if (a.angles) {
#pragma unroll
      for (int e = 0; e < NP; ++e) {
        const float2 x = table[e * a.angles + w * a.items + c];
        cs[e] = x.x;
        sn[e] = x.y;
      }
    } else {
      item_angles<NP>(a.sp, len + i0 + w, c, cs, sn);
    }
    turn<NP>(v, cs, sn, a.sp.interleaved);
  };
  const bool any = i < count;
  Raw<TI, NP> raw{};
  if (any) raw = load(h0, i);
  __shared__ uint32_t part[3][kPageThreads / 32];
  const bool wide = a.dim % 16 == 0 && reinterpret_cast<uintptr_t>(r.out) % 16 == 0;
  const int vecs = a.dim / 16;
  const bool early = wide && old * vecs <= threads;
  for (int h = h0; h < h1; ++h) {
    uint8_t* const head = pool + h * a.dim;
    const float s_old = old ? scales[h] : 0.f;  // (read by all before one of them writes it)
    // Old codes are asked for before it is known whether they are needed: a decode step would wait for them otherwise.
    uint4 codes = make_uint4(0, 0, 0, 0);
    if (early && tid < old * vecs)
      codes = *reinterpret_cast<const uint4*>(head + tid / vecs * pool_row + tid % vecs * 16);
    float v[2 * NP];
    values(raw, any ? i : 0, v);
    if (h + 1 < h1 && any) raw = load(h + 1, i);
    uint32_t amax = 0;  // magnitudes as integers order like the floats; infinities and NaN are above them
    if (any) {
#pragma unroll
      for (int e = 0; e < 2 * NP; ++e) amax = max(amax, __float_as_uint(v[e]) & 0x7fffffffu);
    }
    for (int w = i + step; w < count; w += step) {
      float o[2 * NP];
      values(load(h, w), w, o);
#pragma unroll
      for (int e = 0; e < 2 * NP; ++e) amax = max(amax, __float_as_uint(o[e]) & 0x7fffffffu);
    }
    auto block_max = [&](uint32_t m, uint32_t* at) {
      m = __reduce_max_sync(0xffffffffu, m);
      if (lane == 0) at[tid / 32] = m;
      __syncthreads();
      return __reduce_max_sync(0xffffffffu, lane < threads / 32 ? at[lane] : 0u);
    };
    amax = block_max(amax, part[(h - h0) & 1]);  // (two places in turn: one barrier a head)
    const bool odd = amax >= 0x7f800000u;
    if (odd) {  // the scale goes by the finite ones
      uint32_t m = 0;
      auto finite = [&](float f) { m = fabsf(f) <= FLT_MAX ? max(m, __float_as_uint(f) & 0x7fffffffu) : m; };
      if (any) {
#pragma unroll
        for (int e = 0; e < 2 * NP; ++e) finite(v[e]);
      }
      for (int w = i + step; w < count; w += step) {
        float o[2 * NP];
        values(load(h, w), w, o);
#pragma unroll
        for (int e = 0; e < 2 * NP; ++e) finite(o[e]);
      }
      amax = block_max(m, part[2]);
      __syncthreads();
    }
    const int k = scale_exp<F>(__uint_as_float(amax));
    const float need = pow2(k);
    float s_new = s_old > need ? s_old : need;
    const float inv = 1.f / s_new;
    // int8 has no NaN: a page that was given one has a NaN scale; it stays until the page is begun anew
    if ((!F::kHasNan && odd) || isnan(s_old)) s_new = NAN;
    const bool careful = odd || k == F::kTop;
    auto write = [&](int w, const float* f) {
      uint8_t* row = head + (old + w) * pool_row;
      *reinterpret_cast<Bits<uint8_t, NP>*>(row + it.o1) = codes_of<F, NP>(f, inv, careful);
      if (it.second) *reinterpret_cast<Bits<uint8_t, NP>*>(row + it.o2) = codes_of<F, NP>(f + NP, inv, careful);
    };
    if (any) write(i, v);
    for (int w = i + step; w < count; w += step) {
      float o[2 * NP];
      values(load(h, w), w, o);
      write(w, o);
    }
    if (tid == 0 && !(old && s_new == s_old)) scales[h] = s_new;
    if (!(old && s_new > s_old)) continue;  // (a NaN: the old codes stay)
    const float ratio = s_old / s_new;
    if (wide) {
      for (int w = tid; w < old * vecs; w += threads) {
        uint8_t* at = head + w / vecs * pool_row + w % vecs * 16;
        Vec<uint8_t, 16> c = unpack<uint8_t, 16>(early ? codes : *reinterpret_cast<const uint4*>(at));
#pragma unroll
        for (int e = 0; e < 16; ++e) c.e[e] = F::code(F::value(c.e[e]) * ratio);
        store_vec<uint8_t, 16>(at, c);
      }
    } else {
      for (int w = tid; w < old * a.dim; w += threads) {
        uint8_t* at = head + w / a.dim * pool_row + w % a.dim;
        *at = F::code(F::value(*at) * ratio);
      }
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

template <typename F>
struct Stored {
  using T = F;
  static constexpr bool kCode = false;
  __device__ static float value(F x, float) { return to_f32(x); }
};
template <>
struct Stored<E4m3> {
  using T = uint8_t;
  static constexpr bool kCode = true;
  __device__ static float value(uint8_t x, float scale) { return E4m3::value(x) * scale; }
};
template <>
struct Stored<Int8> {
  using T = uint8_t;
  static constexpr bool kCode = true;
  __device__ static float value(uint8_t x, float scale) { return Int8::value(x) * scale; }
};

// Thread = NV elements of one token's kv head of sequence blockIdx.y, of keys (blockIdx.z 0) or values; positions
// outside the sequence give zeros, and so do those without a page.  Instructions bound it (issue slots 60% busy: four
// integer divisions a thread): int8 prompts 41 us for 165 MB, 25 us of HBM.
template <typename F, typename TO, int NV>
__global__ void __launch_bounds__(256) gather_tokens_kernel(const __grid_constant__ GatherArgs a) {
  using S = typename Stored<F>::T;
  const int s = blockIdx.y, len = a.lens[s];
  const long long start = a.starts ? a.starts[s] : 0ll;
  const unsigned per_tok = (unsigned)a.hk * a.vecs;
  const unsigned w = blockIdx.x * 256u + threadIdx.x;  // (the launch has less than 2^32 of a sequence)
  const unsigned i = w / per_tok, x = w % per_tok;
  const long long pos = start + i;
  if (i >= (unsigned)a.count) return;
  const int h = (int)(x / a.vecs), e = (int)(x % a.vecs) * NV;
  Vec<TO, NV> o;
#pragma unroll
  for (int j = 0; j < NV; ++j) o.e[j] = from_f32<TO>(0.f);
  if (pos >= 0 && pos < len) {
    if (pos / a.bs >= a.max_blocks) {
      atomicCAS(&g_notice, 0, kNoticeTableOverrun);
    } else {
      const int p = (int)pos;
      const long long page = a.table[(long long)s * a.max_blocks + p / a.bs];
      if (page < 0 || page >= a.num_blocks) {  // (freed by a window, or out of range: nothing of the sequence's is there)
        skip_notice();
      } else {
        const S* pool = reinterpret_cast<const S*>(blockIdx.z ? a.v : a.k);
        const Vec<S, NV> in = unpack<S, NV>(
            *reinterpret_cast<const Bits<S, NV>*>(pool + ((page * a.bs + p % a.bs) * a.hk + h) * a.dim + e));
        const float scale = Stored<F>::kCode ? (blockIdx.z ? a.vs : a.ks)[page * a.hk + h] : 1.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) o.e[j] = from_f32<TO>(Stored<F>::value(in.e[j], scale));
      }
    }
  }
  TO* out = reinterpret_cast<TO*>(blockIdx.z ? a.vo : a.ko) + (((long long)s * a.count + i) * a.hk + h) * a.dim + e;
  store_vec<TO, NV>(out, o);
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

// Items of a CTA of `threads` threads: whole tokens (one where a token has more items than that).
static int cta_tokens(int items, int threads) { return items >= threads ? 1 : threads / items; }

// Head lanes of a tensor with these strides in a CTA of `threads` (rotary_kernel).
static int head_lanes(const Rows& r, int heads, int items, int threads = 256) {
  return heads >= 4 && items * 4 <= threads && r.xs[1] < r.xs[2] ? 4 : 1;
}

// Heads per CTA, for `ctas` CTAs of 256 threads that three of an SM hold at a time: one group of all heads (the sines
// are shared) unless that leaves SMs idle; above a wave, few enough groups that the last wave is nearly full (B4 S8192
// Hq32 Hkv8, tokens of a head side by side: 114 us in 2.3 waves, 109 in 6.9; where heads lie side by side, their groups
// would come to the same memory at different times: 112 us in one, 130 in two).  A head for each lane at least.
static int head_group(int ctas, int heads, int lanes) {
  const int wave = 148 * 3, most = heads / lanes > 1 ? heads / lanes : 1;
  int groups = wave / ctas < most ? (wave / ctas > 1 ? wave / ctas : 1) : most;
  for (int g = groups; g <= most && g < groups + 4 && lanes == 1 && ctas > wave / 2; ++g) {
    const double waves = (double)ctas * g / wave;
    if (waves > 1 && (long long)waves + 1 <= 1.06 * waves) {
      groups = g;
      break;
    }
  }
  const int group = (heads + groups - 1) / groups;
  const int least = (heads + 65534) / 65535;  // (a grid dimension)
  return (group + lanes - 1) / lanes * lanes > least ? (group + lanes - 1) / lanes * lanes : least;
}

template <typename T, int NP>
static void launch_rotary(Args& a, cudaStream_t st) {
  const int heads = a.t[0].heads + a.t[1].heads;
  a.items = items_of(NP, a.sp.rot, a.dim);
  a.head_lanes = head_lanes(a.t[a.t[0].heads ? 0 : 1], heads, a.items);
  a.cta_tokens = cta_tokens(a.items * a.head_lanes, 256);
  const int ctas = (a.tokens - 1) / a.cta_tokens + 1;
  a.head_group = head_group(ctas, heads, a.head_lanes);
  const dim3 grid(ctas, (heads + a.head_group - 1) / a.head_group);
  rotary_kernel<T, NP><<<grid, 256, 0, st>>>(a);
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
  if (tokens > INT_MAX - 256) return ATTN_ERR_UNSUPPORTED;
  a.tokens = (int)tokens; a.seq = p->seq; a.dim = p->head_dim;
  const int es = (int)dtype_size(p->dtype);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto ok = [&](int np) {
    if (a.sp.rot / 2 % np || a.dim % np) return false;
    for (const Rows& r : a.t)
      if (r.heads && !(fits(r.x, r.xs, es, np * es) && fits(r.out, r.os, es, np * es))) return false;
    return true;
  };
#define LAUNCH(T, NP) launch_rotary<T, NP>(a, st)
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
  if (bits8 && (long long)p->block_size * p->num_heads_kv > INT_MAX / p->head_dim)
    return ATTN_ERR_UNSUPPORTED;  // (a page's offsets are 32 bits)
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
  if (tokens > INT_MAX - 256) return ATTN_ERR_UNSUPPORTED;
#define WIDE(TI, TO, NP)                                                               \
  do {                                                                                 \
    a.items = items_of(NP, a.sp.rot, a.dim);                                           \
    const int heads = a.q.heads + 2 * a.k.heads;                                       \
    a.head_lanes = head_lanes(a.k, heads, a.items);                                    \
    a.cta_tokens = cta_tokens(a.items * a.head_lanes, 256);                            \
    const int ctas = (int)((tokens - 1) / a.cta_tokens + 1);                           \
    a.head_group = head_group(ctas, heads, a.head_lanes);                              \
    const dim3 grid(ctas, (heads + a.head_group - 1) / a.head_group); \
    append_kernel<TI, TO, NP><<<grid, 256, 0, st>>>(a);                                \
  } while (0)
#define BITS8(TI, F, NP)                                                               \
  do {                                                                                 \
    a.items = items_of(NP, a.sp.rot, a.dim);                                           \
    a.page_slots = (int)(((long long)a.num_new + a.bs - 1) / a.bs) + 1;                \
    if (a.items > kPageThreads) return ATTN_ERR_UNSUPPORTED;                           \
    const long long most = ll_min(a.num_new, a.bs) * (long long)a.items;               \
    const int threads = (int)ll_min(kPageThreads, ll_max(128, (most + 31) / 32 * 32)); \
    a.angles = a.sp.rot && most * NP * 8 <= kAngleBytes ? (int)most : 0;               \
    a.head_lanes = head_lanes(a.q, a.q.heads, a.items, threads);                       \
    a.cta_tokens = cta_tokens(a.items * a.head_lanes, threads);                        \
    a.q_ctas = (int)((tokens + a.cta_tokens - 1) / a.cta_tokens);                      \
    a.head_group = a.q.heads ? head_group(a.q_ctas, a.q.heads, a.head_lanes) : 1;                 \
    const long long groups = (a.q.heads + a.head_group - 1) / a.head_group;            \
    const long long slots = (long long)a.num_seqs * a.page_slots * 2;                  \
    /* heads of a CTA: as many as leave about 16 CTAs per SM */                        \
    a.page_heads = (int)ll_max(1, ll_min(a.k.heads, slots * a.k.heads / (148 * 16)));   \
    const long long pages = slots * ((a.k.heads + a.page_heads - 1) / a.page_heads);   \
    if (pages + a.q_ctas * groups > INT_MAX) return ATTN_ERR_UNSUPPORTED;              \
    a.page_ctas = (int)pages;                                                          \
    append8_kernel<TI, F, NP><<<(unsigned)(pages + a.q_ctas * groups), threads, a.angles * NP * 8, st>>>(a); \
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
  const bool wider = bits8 && a.dim % 16 == 0 && (in | out) % 16 == 0;
  if (a.num_seqs > 65535) return ATTN_ERR_UNSUPPORTED;  // (a grid dimension)
#define RUN(F, TO, NV)                                                                 \
  do {                                                                                 \
    a.vecs = a.dim / NV;                                                               \
    const long long n = ((long long)a.count * a.hk * a.vecs + 255) / 256;              \
    if (n > (1 << 24) - 1) return ATTN_ERR_UNSUPPORTED;                                \
    gather_tokens_kernel<F, TO, NV><<<dim3((unsigned)n, a.num_seqs, 2), 256, 0, st>>>(a); \
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
#define W8(F)               \
  do {                      \
    if (wider) TO_(F, 16);  \
    else W(F);              \
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
