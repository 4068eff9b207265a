// Attention over the 8-bit block cache on tcgen05, for calls with more than 32 query rows per kv head (kv8.cuh has the
// cache's layout and the warp-level kernel for fewer).
//
// A CTA takes up to 64 query rows (r = t * group + j) of one kv head and a run of 128-key tiles (4 pages). The tensor
// cores read fp16, so the codes become fp16 tiles in shared memory first, exactly (the scales stay outside):
//   warps 0-3 (warpgroup 0) and 4-7 (warpgroup 1): softmax of the even and the odd tiles;
//   warps 8-11: page w of each tile, K: bulk copies of header and K into the warp's own ring, codes -> K tile;
//   warps 12-15: the same for V;
//   warp 16: issues Q K^T, warp 17: issues P V. (One warp for both took 1980 cycles a tile: some 65 for each of 16 MMAs, and
//   the waits between them.)
// S = Q K^T as in verify.cuh: M = 64 accumulators, the tile's two 64-key halves at lane offsets 0 and 16, so a lane
// scores 64 keys (two pages) of one row and no lane is padding. With one factor per page, a lane needs two multipliers
// for its 64 scores; the V scale goes into the exponent (see kv8_softmax). Each (warpgroup, half) keeps its own running
// (max, sum, O); the four streams meet at the end. With the two warpgroups on alternate tiles one's TMEM loads, maxima
// and stores run beside the other's exponentials.
//
// What bounds it: a tile (16.5 KB, 710 cycles of an SM's share of HBM) takes about 1700 cycles at head_dim 64. A timeline
// of one CTA puts 1850 on a warpgroup's softmax of every other tile, 1300-1600 on a converter's tile, 8 MMAs of some 70
// cycles on each issuing warp, all on 4.5 warps per scheduler; shared memory alone moves 144 KB a tile, 1150 cycles (codes
// in, codes out, fp16 in, operands out). The warp-level kernel converts in registers and has no such traffic, but its
// MMAs (8 cycles each per scheduler, 1024 a tile at 64 rows) and 4 times the conversions come to more from 33 rows on.
// Measured: 16 tokens over 131072 at 32/8/64 (int8) 59.1 us with the merge (2.3 TB/s), against 92 for the other kernel.
// The order of keys within a page is free as long as P and V agree: V's 16-byte row c of a dim holds the keys 2c, 2c + 1,
// 2c + 8, 2c + 9, 16 + 2c, 17 + 2c, 24 + 2c, 25 + 2c, which is how a lane finds them in the cache.
#pragma once
#include "kv8.cuh"

namespace lfm3a {

constexpr int kTcTile = 128;                                   // keys per tile
constexpr int kTcThreads = 18 * 32;
template <int D>
struct Kv8Tc {
  static constexpr int kStages = D == 64 ? 4 : 2;              // raw ring of a converter warp
  // fp16 tiles of K and of V. V's are what the pipeline turns on: PV(j) frees a tile, a converter takes some 1300 cycles to
  // fill it again.
  static constexpr int kKBufs = D == 64 ? 2 : 1, kVBufs = D == 64 ? 4 : 2;
  static constexpr int kRawK = Q8Section<D>::kOffV;            // header and K codes
  static constexpr int kRawV = 32 * D;
  static constexpr int kPage = 64 * D;                         // a page's K or V as fp16
  static constexpr int kTileBytes = 4 * kPage;
  static constexpr int kPBuf = 16384;                          // [half] 64 rows x 64 keys fp16
  static constexpr int kOffK = 128 * D;                        // after Q: 64 rows x D fp16
  static constexpr int kOffV = kOffK + kKBufs * kTileBytes;
  static constexpr int kOffP = kOffV + kVBufs * kTileBytes;
  static constexpr int kOffRawK = kOffP + 2 * kPBuf;
  static constexpr int kOffRawV = kOffRawK + 4 * kStages * kRawK;
  static constexpr int kOffScale = kOffRawV + 4 * kStages * kRawV;   // [tile % 8][page] (K factor, log2 V factor, 1 / it)
  static constexpr int kOffML = kOffScale + 32 * 16;                 // warpgroup 1's (max, sum, sum of rounded P) per lane
  static constexpr int kOffBar = kOffML + 128 * 16;
  static constexpr int kBars = 8 * kStages + kKBufs + kVBufs + 16 + 2 + 2;
  static constexpr int kOffTmemSlot = kOffBar + kBars * 8;
  static constexpr int kOffAbort = kOffTmemSlot + 4;
  static constexpr int kSmem = kOffAbort + 4;
  static constexpr uint32_t kTmemCols = D == 64 ? 256 : 512;   // S[tile % 2] at 64 (tile % 2), O_g at 128 + D g
  static constexpr uint32_t kSbo = 16 * D;                     // bytes between 8-row groups of Q and K
  static constexpr uint32_t kIdescPV = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((64u >> 4) << 24);   // M64 N = D
};

template <int D, bool E4M3>
__global__ __launch_bounds__(kTcThreads, 1) void kv8_attend_tc_kernel(Kv8AttnArgs a) {
  using L = Kv8Tc<D>;
  using S = Q8Section<D>;
  constexpr int NS = L::kStages, NK = L::kKBufs, NV = L::kVBufs;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  float4* sScale = reinterpret_cast<float4*>(smem + L::kOffScale);
  float4* sML = reinterpret_cast<float4*>(smem + L::kOffML);
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(smem + L::kOffBar);   // [converter warp][stage]
  uint64_t* k_full = raw_full + 8 * NS;
  uint64_t* v_full = k_full + NK;
  // QK of tile i is done: s_full[i & 7]; PV: pv_done[i & 7]. Eight of each, so that whoever waits for tile i knows tile i - 8
  // done and tile i + 8 not: a parity says no more than that.
  uint64_t* s_full = v_full + NV;
  uint64_t* pv_done = s_full + 8;
  uint64_t* p_full = pv_done + 8;    // [tile & 1]
  uint64_t* q_ready = p_full + 2;
  uint64_t* drain = q_ready + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffTmemSlot);
  int& s_abort = *reinterpret_cast<int*>(smem + L::kOffAbort);
  auto aborted = [&] { return __any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(&s_abort) != 0); };

  auto wait_tile = [&](uint64_t* bars, int i) {
    return __all_sync(0xffffffffu, mbar_wait(&bars[i & 7], (uint32_t)(i >> 3) & 1u));
  };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y, split = blockIdx.x, row0 = blockIdx.z * 64, rows = a.m * a.group;
  const int kv_end = a.ctx_len + a.m;
  // The split's tiles of [p_begin / 4, last page / 4].
  const int t_begin = a.p_begin / 4, t_total = (a.p_begin + a.p_total - 1) / 4 - t_begin + 1;
  const int tile0 = t_begin + (int)((int64_t)t_total * split / a.splits);
  const int ntiles = t_begin + (int)((int64_t)t_total * (split + 1) / a.splits) - tile0;

  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < 8 * NS; ++i) mbar_init(&raw_full[i], 1);
    for (int i = 0; i < NK; ++i) mbar_init(&k_full[i], 4);
    for (int i = 0; i < NV; ++i) mbar_init(&v_full[i], 4);
    for (int i = 0; i < 8; ++i) {
      mbar_init(&s_full[i], 2);
      mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&p_full[i], 4);
    mbar_init(q_ready, 8);
    mbar_init(drain, 2);
    fence_barrier_init();
  }
  // A programmatic dependent: nothing global is touched, and no TMEM taken, before the previous kernel has completed.
  pdl_wait();
  if (warp == 16) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 8) {
    // ================================================================ softmax: warpgroup g takes the tiles j = g (mod 2)
    const int g = warp >> 2, quad = warp & 3, hh = lane >> 4;
    const int rr = 16 * quad + (lane & 15), r = row0 + rr;   // this lane's query row
    const bool row_ok = r < rows, warp_ok = row0 + 16 * quad < rows;
    const int t = r / a.group, qpos = a.ctx_len + t;
    const int row = t * a.q_heads + h * a.group + (r - t * a.group);
    // Q: the two warpgroups and halves take a quarter of the row's chunks each. The K tile holds int8 codes with their bias
    // (decode_raw: one instruction per pair), which comes to a constant per row.
    float bias = 0.f;
    if (!E4M3 && row_ok) {
      const uint4* src = reinterpret_cast<const uint4*>(a.q + t * a.q_stride + (int64_t)(h * a.group + (r - t * a.group)) * D);
#pragma unroll 4
      for (int i = 0; i < D / 8; ++i) {
        const uint4 v = src[i];
        const float2 s0 = fadd2(unpack_half2(v.x), unpack_half2(v.y)), s1 = fadd2(unpack_half2(v.z), unpack_half2(v.w));
        bias += (s0.x + s0.y) + (s1.x + s1.y);
      }
      bias *= -kCodeBias<E4M3>;
    }
    {
      const uint4* src = reinterpret_cast<const uint4*>(a.q + t * a.q_stride + (int64_t)(h * a.group + (r - t * a.group)) * D);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int c = (2 * g + hh) * (D / 32) + i;
        *reinterpret_cast<uint4*>(sQ + ((rr >> 3) * (D / 8) + c) * 128 + (rr & 7) * 16) =
            row_ok ? src[c] : make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
    }
    const uint32_t lane_base = tmem + ((uint32_t)(32 * quad) << 16);
    const uint32_t o_col = 128 + D * g;
    uint8_t* pb = smem + L::kOffP + g * L::kPBuf + hh * 8192 + (rr >> 3) * 1024 + (rr & 7) * 16;
    float m_run = -INFINITY, l_run = 0.f, lp_run = 0.f;
    bool ok = true;
    for (int jt = g; jt < ntiles && ok; jt += 2) {
      if (!wait_tile(s_full, jt)) {
        raise_error(kErrWaitMma);
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t s_col = 64 * g;
      if (warp_ok) {
        float4 sc0 = sScale[(jt & 7) * 4 + 2 * hh], sc1 = sScale[(jt & 7) * 4 + 2 * hh + 1];
        if (!E4M3) {   // .w: whether the page holds biased codes (an open page does not)
          sc0.y = fmaf(sc0.w * bias, sc0.x, sc0.y);
          sc1.y = fmaf(sc1.w * bias, sc1.x, sc1.y);
        }
        const int k0 = (tile0 + jt) * kTcTile + 64 * hh;
        const bool open = k0 + 63 <= a.ctx_len && (a.window == 0 || k0 > kv_end - 1 - a.window);
        const int lo = (a.window > 0 ? qpos - a.window + 1 : 0) - k0, hi = qpos - k0;
        float x[32];
        auto load_page = [&](int p) {   // the scores of the lane's page p, masked
          uint32_t u[2][16];
          tmem_ld16(lane_base + s_col + 32 * p, u[0]);
          tmem_ld16(lane_base + s_col + 32 * p + 16, u[1]);
          tmem_wait_ld();
          reg_fence16(u[0]);
          reg_fence16(u[1]);
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(u[i >> 4][i & 15]);
          if (!open) {
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] = 32 * p + k >= lo && 32 * p + k <= hi ? x[k] : -INFINITY;
          }
        };
        // Page 0 is read twice: once for the maximum, once for its exponentials (64 scores at once would spill).
        load_page(0);
        float mx = fmaf(max32(x), sc0.x, sc0.y);
        load_page(1);
        mx = fmaxf(mx, fmaf(max32(x), sc1.x, sc1.y));
        // P_g and O_g are free once PV(jt - 2) is done.
        if (jt >= 2 && !wait_tile(pv_done, jt - 2)) {
          raise_error(kErrWaitMma);
          ok = false;
          break;
        }
        tc_fence_after();
        const bool grow = mx > m_run + (kLazy + kHeadroom);
        if (__any_sync(0xffffffffu, grow)) {
          const float corr = grow ? fast_exp2(m_run - (mx - kHeadroom)) : 1.f;
          if (grow) m_run = mx - kHeadroom;
          l_run *= corr;
          lp_run *= corr;
          if (jt >= 2) {
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(lane_base + o_col + 16 * c, o);
              tmem_wait_ld();
              reg_fence16(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
              tmem_st16(lane_base + o_col + 16 * c, o);
            }
            tmem_wait_st();
          }
        }
        const float neg = m_run == -INFINITY ? 0.f : -m_run;
        auto exp_page = [&](int p, const float4& sc) {
          const float2 kf = make_float2(sc.x, sc.x), off = make_float2(sc.y + neg, sc.y + neg);
          float2 ls = make_float2(0.f, 0.f), lps = ls;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {   // keys 8 i + 2 c and the next
              const int k = 8 * i + 2 * c;
              const float2 e = ffma2(make_float2(x[k], x[k + 1]), kf, off);
              const float2 pr = make_float2(fast_exp2(e.x), fast_exp2(e.y));
              const float2 rr = round11(pr);
              ls = fadd2(ls, pr);
              w[i] = pack_half2(rr.x, rr.y);
              lps = fadd2(lps, rr);
            }
            *reinterpret_cast<uint4*>(pb + (4 * p + c) * 128) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          l_run = fmaf(ls.x + ls.y, sc.z, l_run);
          lp_run = fmaf(lps.x + lps.y, sc.z, lp_run);
        };
        exp_page(1, sc1);
        load_page(0);
        exp_page(0, sc0);
        fence_proxy_async_smem();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[g]);
    }
    if (!ok) atomicExch(&s_abort, 1);
    if (g == 1) sML[32 * quad + lane] = make_float4(m_run, l_run, lp_run, 0.f);
    // The last MMAs (all of both warpgroups' PV): then both O_g of a row, and its two halves, meet.
    const bool done = __all_sync(0xffffffffu, mbar_wait(drain, 0));
    if (!done) {
      raise_error(kErrWaitMma);
      atomicExch(&s_abort, 1);
    }
    named_bar_sync(1, 256);
    if (g == 0 && done && warp_ok && !aborted()) {
      tc_fence_after();
      const float4 b = sML[32 * quad + lane];
      // acc / lp is the mean over rounded P (round11); relative to the exact sums from here on
      const float n0 = lp_run > 0.f ? l_run / lp_run : 1.f, n1 = b.z > 0.f ? b.y / b.z : 1.f;
      float M = fmaxf(m_run, b.x);
      M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 16));
      const float e0 = m_run == -INFINITY ? 0.f : fast_exp2(m_run - M), e1 = b.x == -INFINITY ? 0.f : fast_exp2(b.x - M);
      float sum = e0 * l_run + e1 * b.y;
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      const float f0 = e0 * n0, f1 = e1 * n1;
      const bool direct = a.splits == 1;
      const float scale = direct && row_ok ? (sum > 0.f ? 1.f / sum : 0.f) * sigmoid_gate(a.gate, row) : 1.f;
      float* part = direct ? nullptr : a.part + ((int64_t)row * a.splits + split) * (D + 2);
#pragma unroll 1
      for (int c = 0; c < D / 16; ++c) {
        uint32_t r0[16], r1[16];
        tmem_ld16(lane_base + 128 + 16 * c, r0);
        tmem_ld16(lane_base + 128 + D + 16 * c, r1);
        tmem_wait_ld();
        reg_fence16(r0);
        reg_fence16(r1);
        float o[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {   // a stream without a key has a factor of 0 and an O that was never written
          o[e] = (f0 > 0.f ? f0 * __uint_as_float(r0[e]) : 0.f) + (f1 > 0.f ? f1 * __uint_as_float(r1[e]) : 0.f);
          o[e] = (o[e] + __shfl_xor_sync(0xffffffffu, o[e], 16)) * scale;
        }
        if (row_ok && hh == 0) {
          if (direct) {
            uint4* dst = reinterpret_cast<uint4*>(a.out + (int64_t)row * D + 16 * c);
#pragma unroll
            for (int q = 0; q < 2; ++q)
              dst[q] = make_uint4(pack_half2(o[8 * q], o[8 * q + 1]), pack_half2(o[8 * q + 2], o[8 * q + 3]),
                                  pack_half2(o[8 * q + 4], o[8 * q + 5]), pack_half2(o[8 * q + 6], o[8 * q + 7]));
          } else {
#pragma unroll
            for (int e = 0; e < 16; e += 2) *reinterpret_cast<float2*>(part + 16 * c + e) = make_float2(o[e], o[e + 1]);
          }
        }
      }
      if (row_ok && hh == 0) {
        if (!direct) *reinterpret_cast<float2*>(part + D) = make_float2(M, sum);
        else if (a.lse) a.lse[row] = (M + log2f(sum)) * kLn2;
      }
    }
  } else if (warp < 16) {
    // ================================================================ converters: page `pg` of each tile, K or V
    const bool is_v = warp >= 12;
    const int pg = warp & 3, cw = warp - 8;
    uint8_t* ring = smem + (is_v ? L::kOffRawV + pg * NS * L::kRawV : L::kOffRawK + pg * NS * L::kRawK);
    const uint32_t raw_bytes = is_v ? L::kRawV : L::kRawK;
    uint64_t* full = raw_full + cw * NS;
    uint64_t* out_full = is_v ? v_full : k_full;
    const int sealed_pages = a.sealed / kBlockTokens, last_page = a.p_begin + a.p_total - 1;
    const char* head = a.g.pool + h * a.g.head_bytes + (is_v ? S::kOffV : 0);
    const TailView tail = tail_of(a.tail, a.g.kv_heads, h, D);
    // This warp's sealed pages are the tiles [j0, j1) of the split.
    const int first_page = tile0 * 4 + pg;
    const int j0 = first_page >= a.p_begin ? 0 : (a.p_begin - first_page + 3) / 4;
    const int limit = min(sealed_pages, last_page + 1);
    const int j1 = min(ntiles, first_page >= limit ? 0 : (limit - first_page + 3) / 4);
    // Table entries 32 at a time, one per lane: entries of the tiles tab0 .. tab0 + 31.
    int tab0 = j0;
    int64_t entry = 0;
    auto load_entries = [&] {
      const int j = tab0 + lane;
      entry = j < j1 ? phys_block(a.g, first_page + 4 * j) : 0;
    };
    load_entries();
    int issued = j0;
    auto issue = [&] {   // the next sealed page, by lane 0
      if (issued - tab0 == 32) {
        tab0 += 32;
        load_entries();
      }
      const int64_t blk = __shfl_sync(0xffffffffu, entry, issued - tab0);
      const int st = (issued - j0) % NS;
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[st], raw_bytes);
        bulk_g2s(ring + st * raw_bytes, head + blk * a.g.block_bytes, raw_bytes, &full[st]);
      }
      ++issued;
    };
    while (issued < j1 && issued - j0 < NS) issue();
    int taken = j0;   // sealed pages whose copies have been waited for
    // Conflict-free both ways: 8 lanes of a phase read 8 chunks of distinct banks and write 8 rows of one tile.
    const int g = lane & 7, c = ((g >> 1) + (lane >> 3)) & 3;
    bool ok = true;
    for (int jt = 0; jt < ntiles && ok; ++jt) {
      const int nb = is_v ? NV : NK, buf = is_v ? jt % NV : jt % NK, page = first_page + 4 * jt;
      // The buffer's last reader.
      if (jt >= nb && !wait_tile(is_v ? pv_done : s_full, jt - nb)) {
        raise_error(kErrWaitEmpty);
        ok = false;
        break;
      }
      uint8_t* dst = smem + (is_v ? L::kOffV : L::kOffK) + buf * L::kTileBytes + pg * L::kPage;
      float4 scale = make_float4(a.qk_scale, 0.f, 1.f, 0.f);
      if (jt >= j0 && jt < j1) {
        const int st = (jt - j0) % NS;
        if (!__all_sync(0xffffffffu, mbar_wait(&full[st], (uint32_t)((jt - j0) / NS) & 1u))) {
          raise_error(kErrWaitFull);
          ok = false;
          break;
        }
        ++taken;
        const uint8_t* src = ring + st * raw_bytes;
        if (!is_v) {
          const float ks = reinterpret_cast<const float*>(src)[0] * kCodeUnit<E4M3>;
          const float vs = reinterpret_cast<const float*>(src)[kFactorWord];
          scale = make_float4(ks * a.qk_scale, __log2f(vs), __fdividef(1.f, vs), 1.f);
          const uint4* k4 = reinterpret_cast<const uint4*>(src + S::kOffK);
#pragma unroll
          for (int s = 0; s < 4 * (D / 64); ++s) {   // 8 keys (s / (D / 64)) x 64 dims
            const uint4 w = k4[s * 32 + g * 4 + c];
            uint4* o = reinterpret_cast<uint4*>(dst + ((s / (D / 64)) * (D / 8) + (s % (D / 64)) * 8 + 2 * c) * 128 + g * 16);
            o[0] = make_uint4(decode_raw<E4M3, false>(w.x), decode_raw<E4M3, true>(w.x), decode_raw<E4M3, false>(w.y),
                              decode_raw<E4M3, true>(w.y));
            o[8] = make_uint4(decode_raw<E4M3, false>(w.z), decode_raw<E4M3, true>(w.z), decode_raw<E4M3, false>(w.w),
                              decode_raw<E4M3, true>(w.w));
          }
        } else {
          const uint4* v4 = reinterpret_cast<const uint4*>(src);
#pragma unroll
          for (int d = 0; d < D / 32; ++d) {   // 4 dims (8 apart) x 8 keys per lane
            const uint4 lo = v4[d * 32 + g * 4 + c], hi = v4[(D / 32 + d) * 32 + g * 4 + c];
            const uint32_t w0[4] = {lo.x, lo.y, lo.z, lo.w}, w1[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<uint4*>(dst + ((4 * d + e) * 4 + c) * 128 + g * 16) =
                  make_uint4(decode_pair<E4M3, false>(w0[e]), decode_pair<E4M3, true>(w0[e]), decode_pair<E4M3, false>(w1[e]),
                             decode_pair<E4M3, true>(w1[e]));
          }
        }
        __syncwarp();   // every lane has read the stage
        if (issued < j1) issue();
      } else {
        // An open page from the tail, or a page outside the keys (zeros: its scores are masked, its V is finite).
        const int t0 = page * kBlockTokens, live = page >= sealed_pages && page <= last_page ? kv_end - t0 : 0;
        if (!is_v) {
          for (int i = lane; i < 4 * D; i += 32) {   // 16-byte rows: 8 dims of a key
            const int key = (i / D) * 8 + (i & 7), d8 = (i % D) >> 3;
            *reinterpret_cast<uint4*>(dst + i * 16) =
                key < live ? *reinterpret_cast<const uint4*>(tail.k + (int64_t)((t0 + key) % kTailTokens) * D + d8 * 8)
                           : make_uint4(0, 0, 0, 0);
          }
        } else {
          for (int i = lane; i < 4 * D; i += 32) {
            const int d = (i >> 5) * 8 + (i & 7), cc = (i >> 3) & 3;
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int key = 8 * k + 2 * cc;
              w[k] = key < live ? tail_v_pair(tail, t0 + key, d, kv_end) : 0u;
            }
            *reinterpret_cast<uint4*>(dst + i * 16) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (!is_v && lane == 0) sScale[(jt & 7) * 4 + pg] = scale;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&out_full[buf]);
    }
    if (!ok) atomicExch(&s_abort, 1);
    // Copies still landing after an early exit (bounded).
    for (; taken < issued; ++taken) (void)mbar_wait(&full[(taken - j0) % NS], (uint32_t)((taken - j0) / NS) & 1u);
  } else if (warp == 16) {
    // ================================================================ Q K^T (the whole warp loops, lane 0 issues)
    bool ok = __all_sync(0xffffffffu, mbar_wait(q_ready, 0));
    if (!ok) raise_error(kErrWaitOther);
    const uint64_t q_desc = umma_desc(smem_u32(sQ), 128, L::kSbo);
    for (int jt = 0; jt < ntiles && ok; ++jt) {
      const int buf = jt % NK;
      if (!__all_sync(0xffffffffu, mbar_wait(&k_full[buf], (uint32_t)(jt / NK) & 1u))) {
        raise_error(kErrWaitFull);
        ok = false;
        break;
      }
      // The softmax of tile jt - 2 has read S_g.
      if (jt >= 2 && !__all_sync(0xffffffffu, mbar_wait(&p_full[jt & 1], (uint32_t)((jt >> 1) - 1) & 1u))) {
        raise_error(kErrWaitOther);
        ok = false;
        break;
      }
      tc_fence_after();
      if (lane == 0) {
        const uint64_t k_desc = umma_desc(smem_u32(smem + L::kOffK + buf * L::kTileBytes), 128, L::kSbo);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)   // keys 64 hh ..: two pages on; lanes + 16 hh
            umma_f16_ss(tmem + ((uint32_t)(16 * hh) << 16) + 64 * (jt & 1), q_desc + 16 * ks,
                        k_desc + (2 * L::kPage >> 4) * hh + 16 * ks, kIdescF16M64N64, ks > 0 ? 1u : 0u);
        umma_commit(&s_full[jt & 7]);
        mbar_arrive(&s_full[jt & 7]);   // passes the converters' scales on, as this thread saw them
      }
      __syncwarp();
    }
    if (!ok) atomicExch(&s_abort, 1);
    if (lane == 0) umma_commit(drain);
    __syncwarp();
    mbar_wait(drain, 0);
  } else {
    // ================================================================ P V
    bool ok = true;
    for (int jt = 0; jt < ntiles && ok; ++jt) {
      const int buf = jt % NV, b = jt & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&v_full[buf], (uint32_t)(jt / NV) & 1u))) {
        raise_error(kErrWaitFull);
        ok = false;
        break;
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&p_full[b], (uint32_t)(jt >> 1) & 1u))) {
        raise_error(kErrWaitOther);
        ok = false;
        break;
      }
      tc_fence_after();
      if (lane == 0) {
        const uint64_t v_desc = umma_desc(smem_u32(smem + L::kOffV + buf * L::kTileBytes), 128, 512);
        const uint64_t p_desc = umma_desc(smem_u32(smem + L::kOffP + b * L::kPBuf), 128, 1024);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)   // 16 keys: half a page
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
            umma_f16_ss(tmem + ((uint32_t)(16 * hh) << 16) + 128 + D * b, p_desc + 512 * hh + 16 * ks,
                        v_desc + (L::kPage >> 4) * (2 * hh + (ks >> 1)) + 16 * (ks & 1), L::kIdescPV,
                        (jt >= 2 || ks > 0) ? 1u : 0u);
        umma_commit(&pv_done[jt & 7]);
      }
      __syncwarp();
    }
    if (!ok) atomicExch(&s_abort, 1);
    if (lane == 0) umma_commit(drain);   // also what the softmax warps wait for before they read O
    __syncwarp();
    mbar_wait(drain, 0);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kTmemCols);
  }
}

}  // namespace lfm3a
