// Attention over 8-bit pages for many rows per kv head (drafts, chunks of a prompt), on tcgen05.  Included by attend8.cu.
//
// Up to two tiles of 128 rows share every K/V tile of 128 tokens.  TMA brings the codes of a tile's pages into a
// two-stage ring; a warpgroup turns them into fp16 (exact) in the swizzled tiles that the products read, once for all
// rows of the CTA; S = Q K^T and O += P V run in TMEM as in the 16-bit kernels, and a thread per row keeps the same two
// maxima and carries the value scales in P as the kernel for few rows does (see there).
//
// What bounds it: a tile takes 3.7 us with two row tiles (3.0 with one), of which the products need 1.8 at the
// sustained rate; the softmax of a row tile takes 2.1 to 2.7 (S is read from TMEM twice, since half of 512 threads
// cannot hold 128 columns each; reading it once took as long), the products in its chain 0.8, the conversion of K and V
// 1.2 to 1.5 each beside it.  V has two places, so that the conversion does not wait for P V (4.1 us with one).  A CTA's
// start and end take 14 us (7 until the query is in place; a row is read, and its partials are stored, by one thread).
// Every row group walks to the end of its split and masks: a chunk of a prompt with nothing in front of it does up to
// twice the work that its rows see.
#pragma once

namespace attnb200 {
namespace attend8 {

template <int D>
struct Tc {
  static constexpr int BM = 128, BN = 128;
  static constexpr int KCH = D / 64;
  static constexpr int THREADS = 512;  // warps 0-7 softmax (two row tiles), 8-11 conversion, 12 TMA, 13 MMA, 14 scales, 15 idle
  static constexpr int TILE = KCH * BN * 128;  // 128 rows of fp16
  static constexpr int CODES = BN * D;         // 128 tokens of codes
  static constexpr int STAGES = 2;
  static constexpr int OFF_K = 2 * TILE, OFF_V = OFF_K + TILE, OFF_CODES = OFF_V + 2 * TILE;
  static constexpr int SMEM = OFF_CODES + STAGES * 2 * CODES + 1024;
};

// mbar_wait of a whole warp: one lane waits, then every lane takes the phase.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  bool ok = true;
  if ((threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity, code);
  __syncwarp();
  return __all_sync(0xffffffffu, ok && mbar_try_wait(bar, parity));
}

// Eight channels of the query as floats: 16 bytes, or 32 of fp32.
__device__ __forceinline__ void widen_q(int dtype, const uint4& lo, const uint4& hi, float (&x)[8]) {
  const uint32_t a[4] = {lo.x, lo.y, lo.z, lo.w}, b[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (dtype == ATTN_F32) {
      x[e] = __uint_as_float(a[e]);
      x[4 + e] = __uint_as_float(b[e]);
    } else if (dtype == ATTN_BF16) {
      x[2 * e] = __uint_as_float(a[e] << 16);
      x[2 * e + 1] = __uint_as_float(a[e] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a[e]));
      x[2 * e] = f.x;
      x[2 * e + 1] = f.y;
    }
  }
}

template <class F, int D>
__global__ void __launch_bounds__(512, 1) attend8_tc_kernel(
    const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ Args a) {
  using C = Tc<D>;
  constexpr int BM = C::BM, BN = C::BN;
  const int hk = blockIdx.x / a.row_groups, rg = blockIdx.x % a.row_groups;
  const int split = blockIdx.y, seq = blockIdx.z;
  int ctx = max(a.lens[seq], 0);
  if (ctx > a.max_blocks * (long long)a.bs) {
    ctx = a.max_blocks * a.bs;
    if (threadIdx.x == 0) atomicCAS(&g_notice, 0, kNoticeTableOverrun);
  }
  const int t0 = split * a.chunk;
  if (t0 >= ctx && split) return;
  const int t1 = (int)ll_min(ctx, (long long)t0 + a.chunk);
  if (split == a.splits - 1 && t1 < ctx && threadIdx.x == 0) atomicCAS(&g_notice, 0, kNoticeContextOverrun);
  const int n = (t1 - t0 + BN - 1) / BN;                                     // tiles
  const int row_tiles = min(2, (a.rows - rg * 2 * BM + BM - 1) / BM);
  const int free_until = min(ctx - a.t + 1, t1);  // tokens of this split in front of it are visible to every row

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sb = (raw + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (sb - raw);
  __shared__ uint64_t bars[21];
  __shared__ uint32_t tmem_slot;
  __shared__ float scales[2][16];  // of a tile's eight units: keys, then values
  __shared__ int nan_from[D];      // first token whose value is NaN in a channel, among those not all rows see
  __shared__ int any_nan;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bar0 = smem_u32(bars);
  auto s_full = [&](int x) { return bar0 + 8u * x; };
  auto p_full = [&](int x) { return bar0 + 8u * (2 + x); };
  auto codes_full = [&](int s) { return bar0 + 8u * (4 + s); };
  auto codes_free = [&](int s) { return bar0 + 8u * (6 + s); };
  auto scales_full = [&](int s) { return bar0 + 8u * (8 + s); };
  auto scales_free = [&](int s) { return bar0 + 8u * (17 + s); };
  auto v_full = [&](int s) { return bar0 + 8u * (s ? 19 : 12); };
  auto v_free = [&](int s) { return bar0 + 8u * (s ? 20 : 14); };
  const uint32_t q_full = bar0 + 80, k_full = bar0 + 88, k_free = bar0 + 104,
                 o_done = bar0 + 120, given_up = bar0 + 128;
  if (threadIdx.x == 0) {
    for (int x = 0; x < 2; ++x) {
      mbar_init(s_full(x), 1);
      mbar_init(p_full(x), 4);  // (one arrival per warp)
      mbar_init(v_full(x), 4);
      mbar_init(v_free(x), 1);
      mbar_init(codes_full(x), 1);
      mbar_init(codes_free(x), 4);
      mbar_init(scales_full(x), 1);
      mbar_init(scales_free(x), 4 * row_tiles);  // (the softmax warps of the tiles that are there)
    }
    mbar_init(q_full, 8);
    mbar_init(k_full, 4);
    mbar_init(k_free, 1);
    mbar_init(o_done, 1);
    mbar_init(given_up, 1);
    fence_mbar_init();
    any_nan = 0;
  }
  for (int d = threadIdx.x; d < D; d += C::THREADS) nan_from[d] = INT_MAX;
  if (warp == 13) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  __syncwarp();
  const uint32_t tmem = tmem_slot;

  if (warp >= 12) {
    if (warp == 12) {
      if (lane == 0) {
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
      }
      // lane u loads unit u of a tile (16 tokens of one page); its pool row, or -1
      auto row_of = [&](int i) {
        const int tok = t0 + i * BN + 16 * lane;
        if (lane >= BN / 16 || tok >= t1) return -1;
        bool there;
        const long long page = page_of(a, seq, tok, &there);
        return (int)(page * a.bs + tok % a.bs);
      };
      int row = n > 0 ? row_of(0) : -1, i = 0;
      for (; i < n; ++i) {
        const int s = i % C::STAGES;
        const int next = i + 1 < n ? row_of(i + 1) : -1;
        if (!wait_warp(codes_free(s), ((i / C::STAGES) & 1) ^ 1, kStatusTimeoutLoad)) break;
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, row >= 0)) * 32u * D;
        if (lane == 0) mbar_expect_tx(codes_full(s), bytes);
        __syncwarp();
        if (row >= 0) {
          const uint32_t dst = sb + C::OFF_CODES + s * 2 * C::CODES + lane * 16 * D;
          tma_load_3d(dst, &tm_k, codes_full(s), 0, hk, row);
          tma_load_3d(dst + C::CODES, &tm_v, codes_full(s), 0, hk, row);
        }
        row = next;
      }
      // (every tile's codes are in place before the block ends; where a role gave up nobody else waits for them)
      for (int u = max(i - C::STAGES, 0); u < i; ++u) mbar_drain(codes_full(u % C::STAGES), (u / C::STAGES) & 1);
    } else if (warp == 13 && lane == 0 && n > 0) {
      constexpr uint32_t ID_S = idesc_f16(BM, BN, 0, 0, 0);
      constexpr uint32_t ID_O = idesc_f16(BM, D, 0, 0, 1);
      const uint64_t dQ = sdesc_sw128(sb, 16, 1024);
      const uint64_t dK = sdesc_sw128(sb + C::OFF_K, 16, 1024);
      const uint64_t dV = sdesc_sw128(sb + C::OFF_V, BN * 128, 1024);  // MN-major
      auto issue_s = [&](int x) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_f16(tmem + x * 128, sdesc_add(dQ, x * C::TILE + (k >> 2) * BM * 128 + (k & 3) * 32),
                   sdesc_add(dK, (k >> 2) * BN * 128 + (k & 3) * 32), ID_S, k > 0 ? 1u : 0u);
        umma_commit(s_full(x));
      };
      auto issue_pv = [&](int x, int i) -> bool {
        if (!mbar_wait(p_full(x), i & 1, kStatusTimeoutMma)) return false;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)
          umma_f16_ts(tmem + 256 + x * D, tmem + x * 128 + k * 8, sdesc_add(dV, (i & 1) * C::TILE + k * 16 * 128), ID_O,
                      (i > 0 || k > 0) ? 1u : 0u);
        return true;
      };
      // S of a row tile is issued behind its P V of the tile before, which reads P from the same columns.
      bool ok = mbar_wait(q_full, 0, kStatusTimeoutMma);
      for (int i = 0; ok && i <= n; ++i) {
        if (i > 0) {
          ok = mbar_wait(v_full((i - 1) & 1), ((i - 1) >> 1) & 1, kStatusTimeoutMma) && issue_pv(0, i - 1);
          if (!ok) break;
          if (row_tiles == 1) umma_commit(v_free((i - 1) & 1));
        }
        if (i < n) {
          ok = mbar_wait(k_full, i & 1, kStatusTimeoutMma);
          if (!ok) break;
          tc_fence_after();
          issue_s(0);
        }
        if (row_tiles == 2 && i > 0) {
          ok = issue_pv(1, i - 1);
          if (!ok) break;
          umma_commit(v_free((i - 1) & 1));
        }
        if (i < n) {
          if (row_tiles == 2) issue_s(1);
          umma_commit(k_free);
        }
      }
      if (ok) {
        umma_commit(o_done);
      } else {  // (products in flight end before their memory is given up)
        umma_commit(given_up);
        mbar_drain(given_up, 0);
      }
    } else if (warp == 14) {
      // Lane u or 8 + u: the key or value scale of unit u.  (A warp of its own: its loads follow one another, page and
      // then scale, and held the conversion up for 0.6 us a tile when one of those warps did this.)
      auto scale_of = [&](int i) {
        const int tok = t0 + i * BN + 16 * (lane & 7);
        if (lane >= 16 || i >= n || tok >= t1) return 0.f;
        bool there;
        const long long page = page_of(a, seq, tok, &there);
        return there ? (lane < 8 ? a.ks : a.vs)[page * a.hkv + hk] : NAN;
      };
      float sc = scale_of(0);
      for (int i = 0; i < n; ++i) {
        if (!wait_warp(scales_free(i & 1), ((i >> 1) & 1) ^ 1, kStatusTimeoutLoad)) break;
        if (lane < 16) scales[i & 1][lane] = sc;
        mbar_arrive_warp(scales_full(i & 1));
        sc = scale_of(i + 1);
      }
    }
  } else if (warp >= 8) {
    const int r = threadIdx.x - 256;  // this thread's token of a tile
    for (int i = 0; i < n; ++i) {
      const int s = i % C::STAGES, tok = t0 + i * BN + r;
      if (!wait_warp(codes_full(s), (i / C::STAGES) & 1, kStatusTimeoutLoad)) break;
      const uint32_t codes = sb + C::OFF_CODES + s * 2 * C::CODES;
      bool ok = true;
#pragma unroll 1
      for (int kv = 0; kv < 2; ++kv) {
        ok = wait_warp(kv ? v_free(i & 1) : k_free, ((kv ? i >> 1 : i) & 1) ^ 1, kStatusTimeoutLoad);
        if (!ok) break;
        uint8_t* const tile = smem + (kv ? C::OFF_V + (i & 1) * C::TILE : C::OFF_K) + r * 128;
        const bool there = tok < t1;  // (K behind the split is masked; V there is zero: P is, but 0 * NaN is not)
        if (there || kv) {
          const bool edge = kv && there && tok >= free_until;
#pragma unroll 2
          for (int c = 0; c < D / 16; ++c) {
            uint4 w = make_uint4(0, 0, 0, 0), lo = w, hi = w;
            if (there) w = lds128(codes + kv * C::CODES + place<D>(r, c));
            if (edge && (F::nan_bytes(w.x) | F::nan_bytes(w.y) | F::nan_bytes(w.z) | F::nan_bytes(w.w))) {
              // A NaN that not all rows see is taken out; the rows that see it get it at the end.
              any_nan = 1;
              uint32_t bad[4] = {F::nan_bytes(w.x), F::nan_bytes(w.y), F::nan_bytes(w.z), F::nan_bytes(w.w)};
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (bad[e / 4] >> (8 * (e % 4)) & 1u) atomicMin(&nan_from[16 * c + e], tok);
              w = make_uint4(w.x & ~bad[0], w.y & ~bad[1], w.z & ~bad[2], w.w & ~bad[3]);
            }
            if (there) F::wide16(w, lo, hi);
            uint8_t* const at = tile + (c >> 2) * BN * 128;
            *reinterpret_cast<uint4*>(at + (((2 * (c & 3)) ^ (r & 7)) << 4)) = lo;
            *reinterpret_cast<uint4*>(at + (((2 * (c & 3) + 1) ^ (r & 7)) << 4)) = hi;
          }
        }
        fence_proxy_async_smem();
        mbar_arrive_warp(kv ? v_full(i & 1) : k_full);
      }
      if (!ok) break;
      mbar_arrive_warp(codes_free(s));
    }
  } else {
    const int x_tile = warp >> 2, rl = threadIdx.x & 127;  // row tile, row in it == TMEM lane
    const int r = (rg * 2 + x_tile) * BM + rl;
    const bool there = r < a.rows;
    const long long row0 = ((long long)seq * a.hq + hk * a.group) * a.t;  // the kv head's rows follow one another
    const int last = there ? min(ctx - a.t + r % a.t + 1, t1) : 0;        // last visible position of this split + 1
    bool ok = x_tile < row_tiles;
    float cq = 0.f;
    if (ok) {
      // A row per thread: a power of two is taken out, and fp16 goes into the swizzled tile.  (The loads are behind no
      // branch: what it would move behind itself waits for them one by one.)
      const int elem = a.dtype == ATTN_F32 ? 4 : 2;
      const uint4* const row = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(a.q) +
                                                              (row0 + min(r, a.rows - 1)) * D * elem);
      uint8_t* const tile = smem + x_tile * C::TILE + rl * 128;
      uint4 raw[D / 8];  // (fp32: eight channels' first half)
#pragma unroll
      for (int p = 0; p < D / 8; ++p) raw[p] = row[p * (elem / 2)];
      float big = 0.f;
#pragma unroll
      for (int p = 0; p < D / 8; ++p) {
        float q[8];
        widen_q(a.dtype, raw[p], elem == 4 ? row[2 * p + 1] : raw[p], q);
#pragma unroll
        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(q[e]));
      }
      const int e2 = query_exponent(big);
      const float mul = there ? __uint_as_float((uint32_t)(127 - e2) << 23) : 0.f;
      cq = query_factor(a, big, e2) * F::kUnshift;
#pragma unroll
      for (int p = 0; p < D / 8; ++p) {
        float q[8];
        widen_q(a.dtype, raw[p], elem == 4 ? row[2 * p + 1] : raw[p], q);
        *reinterpret_cast<uint4*>(tile + (p >> 3) * BM * 128 + (((p & 7) ^ (rl & 7)) << 4)) =
            make_uint4(half_pair(q[0] * mul, q[1] * mul), half_pair(q[2] * mul, q[3] * mul),
                       half_pair(q[4] * mul, q[5] * mul), half_pair(q[6] * mul, q[7] * mul));
      }
      fence_proxy_async_smem();
    }
    mbar_arrive_warp(q_full);
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_addr = lanes + x_tile * 128, o_addr = lanes + 256 + x_tile * D;
    // A warp without rows leaves the exponentials to the others; what its lanes of P and O hold reaches no other row.
    const bool idle = r - lane >= a.rows;
    float m = -FLT_MAX, mo = -FLT_MAX, up = 256.f, l = 0.f;
    for (int i = 0; ok && i < n; ++i) {
      const int tok0 = t0 + i * BN;
      ok = wait_warp(scales_full(i & 1), (i >> 1) & 1, kStatusTimeoutSoftmax) &&
           wait_warp(s_full(x_tile), i & 1, kStatusTimeoutSoftmax);
      if (!ok) break;
      tc_fence_after();
      if (idle) {
        tc_fence_before();
        mbar_arrive_warp(scales_free(i & 1));
        mbar_arrive_warp(p_full(x_tile));
        continue;
      }
      const float* ks = scales[i & 1];
      const float* vs = scales[i & 1] + 8;
      const bool whole = tok0 + BN <= free_until;
      // the maximum of the scores in log2, and that of score + log2 of the value scale
      // (64 columns at a time, here and below, in loops that stay rolled: all 128 do not fit a thread's registers.)
      float mx = -FLT_MAX, mxo = -FLT_MAX, lvx = -100.f;
#pragma unroll 1
      for (int c0 = 0; c0 < BN; c0 += 64) {
        float x[64];
#pragma unroll
        for (int c = 0; c < 64; c += 32) tmem_ld32(s_addr + c0 + c, *reinterpret_cast<uint32_t(*)[32]>(&x[c]));
        tmem_wait_ld();
        if (!whole) {
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (tok0 + c0 + c >= last) x[c] = -INFINITY;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float pm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 16 * u; c < 16 * u + 16; ++c) pm[c & 3] = fmaxf(pm[c & 3], x[c]);
          const float top = fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3]));
          const float p = top == -INFINITY ? top : top * (ks[c0 / 16 + u] * cq);  // (scales are not negative)
          mx = fmaxf(mx, p);
          const float lv = fmaxf(lg2(vs[c0 / 16 + u]), -100.f);
          mxo = fmaxf(mxo, p + lv);
          lvx = fmaxf(lvx, lv);
        }
      }
      float fo = 1.f;
      if (mx > m + kSlack || mxo > mo + kSlack) {
        const float m_new = fmaxf(m, mx), mo_new = fmaxf(mo, mxo);
        l *= ex2(m - m_new);
        fo = ex2(mo - mo_new);
        m = m_new;
        mo = mo_new;
        up = ex2(m - mo + kHead);
      }
      unsigned long long sum[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
      auto weights = [&](auto far_units) {
        constexpr bool FAR = decltype(far_units)::value;
        constexpr int W = FAR ? 32 : 64;
        // (S is read again; P, half as wide, stays behind what has been read.)
#pragma unroll 1
        for (int c0 = 0; c0 < BN; c0 += W) {
          float x[W];
#pragma unroll
          for (int c = 0; c < W; c += 32) tmem_ld32(s_addr + c0 + c, *reinterpret_cast<uint32_t(*)[32]>(&x[c]));
          tmem_wait_ld();
          uint32_t pk[W / 2];
#pragma unroll
          for (int u = 0; u < W / 16; ++u) {
            const float f = ks[c0 / 16 + u] * cq;
            float g = vs[c0 / 16 + u] * up, from = -m, in_sum = 1.f;
            if (FAR) {  // (w without p, as in the kernel for few rows)
              const float lv = fmaxf(lg2(vs[c0 / 16 + u]), -100.f);
              const bool far = lv + (m - mo) > kFar;
              g = far ? 256.f : g;
              from = far ? lv - mo : from;
              in_sum = far ? 0.f : 1.f;
            }
            const unsigned long long f2 = f2_pack(f, f), g2 = f2_pack(g, g), nm2 = f2_pack(from, from);
#pragma unroll
            for (int c = 16 * u; c < 16 * u + 16; c += 2) {
              float y0, y1;
              f2_unpack(f2_fma(f2_pack(x[c], x[c + 1]), f2, nm2), y0, y1);
              y0 = ex2(y0);
              y1 = ex2(y1);
              if (!whole) {  // (f may be 0, g NaN)
                if (tok0 + c0 + c >= last) y0 = 0.f;
                if (tok0 + c0 + c + 1 >= last) y1 = 0.f;
              }
              const unsigned long long p = f2_pack(y0, y1);
              sum[(c >> 1) & 1] = FAR ? f2_fma(p, f2_pack(in_sum, in_sum), sum[(c >> 1) & 1]) : f2_add(sum[(c >> 1) & 1], p);
              f2_unpack(f2_mul(p, g2), y0, y1);
              pk[c / 2] = half_pair(y0, y1);
            }
          }
          if (!whole) {
#pragma unroll
            for (int c = 0; c < W; c += 2) {
              if (tok0 + c0 + c >= last) pk[c / 2] = 0u;
              else if (tok0 + c0 + c + 1 >= last) pk[c / 2] &= 0xffffu;
            }
          }
          tmem_st_cols<W / 2>(s_addr + c0 / 2, pk);
        }
      };
      // (a copy of its own: its factors of every unit would not fit the registers of the usual case)
      if (__any_sync(0xffffffffu, lvx + (m - mo) > kFar)) weights(std::true_type{});
      else weights(std::false_type{});
      float s0, s1, s2, s3;
      f2_unpack(sum[0], s0, s1);
      f2_unpack(sum[1], s2, s3);
      l += (s0 + s1) + (s2 + s3);
      // P V of the tile before is complete: S of this one was issued behind it.
      if (i > 0 && __any_sync(0xffffffffu, fo != 1.f)) {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fo);
          tmem_st32(o_addr + c * 32, o);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive_warp(p_full(x_tile));
      mbar_arrive_warp(scales_free(i & 1));
    }
    // (the last V tile's barrier too: what its makers noted about NaN is then seen)
    if (ok && n > 0)
      ok = wait_warp(v_full((n - 1) & 1), ((n - 1) >> 1) & 1, kStatusTimeoutSoftmax) && wait_warp(o_done, 0, kStatusTimeoutSoftmax);
    if (ok) {
      tc_fence_after();
      if (!there) l = 0.f;
      const float inv = l == 0.f ? 0.f : ex2(mo - m - kHead - F::kShift) / l;
      const bool patch = any_nan && l != 0.f;
      const long long at = a.splits == 1 ? row0 + r : (row0 + r) * a.splits + split;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        __syncwarp();
        if (n > 0) {
          tmem_ld32(o_addr + c * 32, o);
          tmem_wait_ld();
        }
        if (!there) continue;
        // (a row without keys may hold o of nothing: select, do not multiply)
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = l == 0.f ? 0u : __float_as_uint(__uint_as_float(o[e]) * inv);
        if (patch) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (nan_from[32 * c + e] < last) o[e] = __float_as_uint(NAN);
        }
        if (a.splits == 1 && a.dtype != ATTN_F32) {
          uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + at * D + c * 32;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = pack2(__uint_as_float(o[8 * v + 2 * e]), __uint_as_float(o[8 * v + 2 * e + 1]), a.dtype == ATTN_BF16);
            *reinterpret_cast<uint4*>(out + 8 * v) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
          float* out = (a.splits == 1 ? reinterpret_cast<float*>(a.out) : a.part_o) + at * D + c * 32;
#pragma unroll
          for (int v = 0; v < 8; ++v)
            *reinterpret_cast<uint4*>(out + 4 * v) = make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
        }
      }
      if (there && a.splits > 1) a.part_lse[(row0 + r) * a.splits + split] = l == 0.f ? -INFINITY : m + lg2(l);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 13) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace attend8
}  // namespace attnb200
