// Eviction from the 8-bit cache by accumulated attention weight: which keys of each kv head stay (evict_select_kernel)
// and their move into a smaller cache (kv8_compact_kernel).
#pragma once
#include "kv8.cuh"

namespace lfm3a {

struct EvictArgs {
  const float* w;        // [kv_heads][stride]
  int32_t* keep;         // [kv_heads][budget], ascending
  float* w_out;          // [kv_heads][out_stride] weights of the kept keys, or null
  int64_t stride, out_stride;
  int len, sink, recent, budget;
  int cached;            // a block's keys fit kEvictCache
};

constexpr int kEvictThreads = 1024;
constexpr int kEvictCache = 48 * 1024;    // keys of a block's share that stay in shared memory
constexpr int kEvictSingle = 16 * 1024;   // positions of a kv head that one block takes

// Weights as unsigned integers of the same order; the zeros are equal and NaN is below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w + 0.f);   // -0 + 0 = +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// A kv head's positions [sink, len - recent) go to a cluster of C blocks, one run each, each of its warps a run of that, in
// order: one block up to 16384 positions, else eight. The k-th largest key is found 8 bits at a time from the top, from
// histograms summed over the cluster's shared memory (every block adds up all of them, so all know the same digit); then
// the warps write the kept positions in order, each starting where the counts of the warps and blocks before it end. Of
// keys equal to the last one kept the first ones stay, so the result does not depend on any order of execution. The keys
// stay in shared memory up to 49152 per block; a longer share is read again (L2) on each sweep. The sweeps are short
// loops: unrolled over registers they were slower, each instruction being fetched for one use. Bound by the latency of its
// steps: 8 heads x 131072 positions take 22.6 us, of which a pass with its cluster barrier is 2.6 (1.9 at 20000), 4 x 5003
// 8.0 us, 8 x 1000 4.9 us.
template <int C>
__device__ __forceinline__ void evict_select(const EvictArgs& a) {
  constexpr int W = kEvictThreads / 32;
  __shared__ __align__(16) uint32_t hist[4][256];
  __shared__ uint32_t found[4][2];     // per pass: the digit, and how many keys lie above it
  __shared__ uint2 warp_count[W];      // per warp: keys above the threshold, and equal to it
  __shared__ uint2 block_count;
  extern __shared__ __align__(1024) uint8_t smem[];
  cg::cluster_group cluster = cg::this_cluster();
  auto sync_all = [&] {
    if constexpr (C > 1) cluster.sync();
    else __syncthreads();
  };
  const int rank = C > 1 ? (int)cluster.block_rank() : 0, h = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = a.len - a.sink - a.recent, k = a.budget - a.sink - a.recent;
  const int i0 = a.sink + (int)((int64_t)n * rank / C);
  const int i1 = a.sink + (int)((int64_t)n * (rank + 1) / C);
  const int run = ((i1 - i0 + kEvictThreads - 1) / kEvictThreads) << 5;   // positions of a warp, whole rows of 32
  const int r0 = min(i1, i0 + warp * run), count = min(i1, r0 + run) - r0;
  (&hist[0][0])[tid] = 0;   // 4 x 256 = the block's threads
  pdl_wait();
  pdl_trigger();
  const float* w = a.w + h * a.stride + r0;
  int32_t* keep = a.keep + (int64_t)h * a.budget;
  float* w_out = a.w_out ? a.w_out + h * a.out_stride : nullptr;
  // This warp's keys; a lane only ever looks at those it put there itself.
  uint32_t* keys = a.cached ? reinterpret_cast<uint32_t*>(smem) + (r0 - i0) : nullptr;
  if (keys) {
#pragma unroll 8
    for (int i = lane; i < count; i += 32) keys[i] = weight_key(w[i]);
  }
  auto key_at = [&](int i) { return keys ? keys[i] : weight_key(w[i]); };
  __syncthreads();   // the histograms are zero
  uint32_t prefix = 0, mask = 0;      // digits found so far
  int left = k;                       // how many of the keys that match the prefix stay
  const bool all = k >= n;
  if (k > 0 && !all) {                // the same in every thread of the cluster
#pragma unroll 1
    for (int pass = 0; pass < 4; ++pass) {
      const int shift = 24 - 8 * pass;
      uint32_t* mine = hist[pass];
#pragma unroll 4
      for (int i = lane; i < count; i += 32) {
        const uint32_t key = key_at(i);
        if ((key & mask) == prefix) atomicAdd(&mine[(key >> shift) & 255u], 1u);
      }
      sync_all();
      if (warp == 0) {   // lane l: the bins 8 l .. 8 l + 7 from the top
        uint32_t own[8] = {};
#pragma unroll
        for (int r = 0; r < C; ++r) {
          const uint4* src = reinterpret_cast<const uint4*>((C > 1 ? cluster.map_shared_rank(mine, r) : mine) + 248 - 8 * lane);
          const uint4 lo = src[0], hi = src[1];
          const uint32_t v[8] = {hi.w, hi.z, hi.y, hi.x, lo.w, lo.z, lo.y, lo.x};
#pragma unroll
          for (int j = 0; j < 8; ++j) own[j] += v[j];
        }
        uint32_t sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += own[j];
        uint32_t incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t u = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += u;
        }
        uint32_t before = incl - sum;
        const uint32_t need = (uint32_t)left;
#pragma unroll
        for (int j = 0; j < 8; ++j) {   // the digit at which the count from the top reaches what is needed
          if (before < need && before + own[j] >= need) {
            found[pass][0] = 255u - (8 * lane + j);
            found[pass][1] = before;
          }
          before += own[j];
        }
      }
      __syncthreads();
      prefix |= found[pass][0] << shift;
      mask |= 255u << shift;
      left -= (int)found[pass][1];
    }
  }

  // Keys above the threshold (all of them when everything stays) and equal to it, of each warp, then before it.
  const uint32_t from = all ? 0u : prefix + 1u;   // prefix < 2^32 - 1: the largest key of a weight is infinity's
  uint32_t gt = 0, eq = 0;
  if (k > 0) {
#pragma unroll 4
    for (int i = lane; i < count; i += 32) {
      const uint32_t key = key_at(i);
      gt += key >= from;
      eq += !all && key == prefix;
    }
  }
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  if (lane == 0) warp_count[warp] = make_uint2(gt, eq);
  __syncthreads();
  const uint2 wc = warp_count[lane];
  uint32_t gt0 = lane < warp ? wc.x : 0u, eq0 = lane < warp ? wc.y : 0u;
  if constexpr (C > 1) {
    if (warp == 0) {
      const uint32_t tg = __reduce_add_sync(0xffffffffu, wc.x), te = __reduce_add_sync(0xffffffffu, wc.y);
      if (lane == 0) block_count = make_uint2(tg, te);
    }
    cluster.sync();
    if (lane < rank) {
      const uint2 c = *cluster.map_shared_rank(&block_count, lane);
      gt0 += c.x;
      eq0 += c.y;
    }
  }
  gt0 = __reduce_add_sync(0xffffffffu, gt0);
  eq0 = __reduce_add_sync(0xffffffffu, eq0);
  if constexpr (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // the counts are read

  if (rank == 0)
    for (int i = tid; i < a.sink; i += kEvictThreads) {
      keep[i] = i;
      if (w_out) w_out[i] = a.w[h * a.stride + i];
    }
  if (rank == C - 1)
    for (int i = tid; i < a.recent; i += kEvictThreads) {
      const int pos = a.len - a.recent + i, at = a.budget - a.recent + i;
      keep[at] = pos;
      if (w_out) w_out[at] = a.w[h * a.stride + pos];
    }
  if (k > 0) {
    const uint32_t below = (1u << lane) - 1u, most = (uint32_t)left;
#pragma unroll 4
    for (int base = 0; base < count; base += 32) {
      const int i = base + lane;
      const uint32_t key = i < count ? key_at(i) : 0u;
      const bool is_gt = i < count && key >= from, is_eq = i < count && !all && key == prefix;
      const uint32_t bg = __ballot_sync(0xffffffffu, is_gt), be = __ballot_sync(0xffffffffu, is_eq);
      const uint32_t my_eq = eq0 + __popc(be & below);
      if (is_gt || (is_eq && my_eq < most)) {
        const int at = a.sink + (int)(gt0 + __popc(bg & below) + min(my_eq, most));
        keep[at] = r0 + i;
        if (w_out) w_out[at] = w[i];
      }
      gt0 += __popc(bg);
      eq0 += __popc(be);
    }
  }
  // No block leaves while another may still read its shared memory.
  if constexpr (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__global__ __launch_bounds__(kEvictThreads) void evict_select_kernel(EvictArgs a) { evict_select<1>(a); }
__global__ __cluster_dims__(8, 1, 1) __launch_bounds__(kEvictThreads) void evict_select_cluster_kernel(EvictArgs a) {
  evict_select<8>(a);
}

struct Kv8CompactArgs {
  KvGeom src, dst;
  __half* src_tail;
  __half* dst_tail;
  const int32_t* keep;   // [kv_heads][budget]
  int len, sealed, budget;
};

// One block per (page of the smaller cache, kv head): the values of its 32 kept tokens (fp32: code times scale, or the
// tail's fp16) are sealed anew under their own scale; an incomplete last page goes to the smaller cache's tail in fp16.
// No value passes through shared memory: a thread makes one chunk of the new page, of K (16 dims of a token, one chunk
// of the old one) or of V (4 dims of 4 tokens: a byte from each word of a chunk of each token's page), and holds it as
// fp16 codes while the block finds the scale. (Staged in shared memory as values it took 67 us for 8 x 32768 of 131072
// tokens, bound by instructions; this takes 36 us, 3.5 TB/s of sectors.)
template <int D, bool E4M3>
__global__ __launch_bounds__(kSealThreads<D>) void kv8_compact_kernel(Kv8CompactArgs a) {
  using S = Q8Section<D>;
  constexpr int U = 2;                      // chunks per thread
  __shared__ __align__(16) float red[16];
  __shared__ const char* sec[32];
  __shared__ int pos[32];
  __shared__ float mult[64];                // what a token's fp16 K and V (codes, or the tail's values) stand for
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, page = blockIdx.x, h = blockIdx.y, t0 = page * kBlockTokens;
  const int live = min(kBlockTokens, a.budget - t0);
  if (tid < 32) {
    const int p = min(max(a.keep[(int64_t)h * a.budget + t0 + min(tid, live - 1)], 0), a.len - 1);
    pos[tid] = p;
    sec[tid] = p < a.sealed ? a.src.pool + phys_block(a.src, p / kBlockTokens) * a.src.block_bytes + h * a.src.head_bytes
                            : nullptr;
  }
  __syncthreads();
  // The scales come beside the chunks, not before them: one round of loads less to wait for.
  float2 f = make_float2(1.f, 1.f);
  if (tid < 32 && sec[tid]) f = *reinterpret_cast<const float2*>(sec[tid]);
  auto publish_scales = [&] {
    if (tid < 32) {
      mult[tid] = sec[tid] ? f.x : 1.f;
      mult[32 + tid] = sec[tid] ? f.y : 1.f;
    }
    named_bar_sync(1, kSealThreads<D>);   // reached from two places
  };
  const TailView from = tail_of(a.src_tail, a.src.kv_heads, h, D), to = tail_of(a.dst_tail, a.dst.kv_heads, h, D);
  const bool is_v = tid >= D;
  uint32_t x[U][8];   // K: dims 2 i, 2 i + 1; V: token b's dims d0, d0 + 8 in x[2 b], d0 + 16, d0 + 24 in x[2 b + 1]
  float kmax = 0.f, vmax = 0.f;
  if (!is_v) {
    uint4 r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = tid + u * D, l = i & 31, c = i >> 5;
      const int t = (c / (D / 64)) * 8 + (l >> 2), d0 = (c % (D / 64)) * 64 + (l & 3) * 16;
      r[u] = make_uint4(0, 0, 0, 0);
      if (sec[t]) r[u] = *reinterpret_cast<const uint4*>(sec[t] + S::kOffK + S::k_chunk(pos[t] % kBlockTokens, d0) * 16);
    }
    publish_scales();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = tid + u * D, l = i & 31, c = i >> 5;
      const int t = (c / (D / 64)) * 8 + (l >> 2), d0 = (c % (D / 64)) * 64 + (l & 3) * 16;
      const uint32_t w[4] = {r[u].x, r[u].y, r[u].z, r[u].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[u][2 * k] = decode_pair<E4M3, false>(w[k]);
        x[u][2 * k + 1] = decode_pair<E4M3, true>(w[k]);
      }
      if (!sec[t]) {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(from.k + (int64_t)(pos[t] % kTailTokens) * D + d0);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[u][k] = src[k];
      }
      __half2 m = __float2half2_rn(0.f);
      m = max_abs8(make_uint4(x[u][0], x[u][1], x[u][2], x[u][3]), m);
      m = max_abs8(make_uint4(x[u][4], x[u][5], x[u][6], x[u][7]), m);
      kmax = fmaxf(kmax, max_of(m) * mult[t]);
    }
  } else {
    uint4 r[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = tid - D + u * D, c = i & 3, g = (i >> 2) & 7, b8 = i >> 5;
      const int dtp = b8 % (D / 32), mt = b8 / (D / 32);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int t = 16 * mt + 2 * c + (b & 1) + 8 * (b >> 1);
        r[u][b] = make_uint4(0, 0, 0, 0);
        if (sec[t])   // the chunk of the old page that holds the token, whatever its byte
          r[u][b] = *reinterpret_cast<const uint4*>(sec[t] + S::kOffV + S::v_index(pos[t] % kBlockTokens & ~9, 32 * dtp + g));
      }
    }
    publish_scales();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = tid - D + u * D, c = i & 3, g = (i >> 2) & 7, b8 = i >> 5;
      const int dtp = b8 % (D / 32), mt = b8 / (D / 32);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int t = 16 * mt + 2 * c + (b & 1) + 8 * (b >> 1), p = pos[t], byte = (p >> 3 & 1) * 2 + (p & 1);
        const uint32_t sel = byte | (4 + byte) << 4;
        x[u][2 * b] = decode_pair<E4M3, false>(__byte_perm(r[u][b].x, r[u][b].y, sel));
        x[u][2 * b + 1] = decode_pair<E4M3, false>(__byte_perm(r[u][b].z, r[u][b].w, sel));
        if (!sec[t]) {
          const uint16_t* src = reinterpret_cast<const uint16_t*>(from.v) + (int64_t)(32 * dtp + g) * kTailTokens + p % kTailTokens;
          x[u][2 * b] = (uint32_t)src[0] | (uint32_t)src[8 * kTailTokens] << 16;
          x[u][2 * b + 1] = (uint32_t)src[16 * kTailTokens] | (uint32_t)src[24 * kTailTokens] << 16;
        }
        const uint32_t a0 = x[u][2 * b] & 0x7fff7fffu, a1 = x[u][2 * b + 1] & 0x7fff7fffu;
        vmax = fmaxf(vmax, max_of(__hmax2(*reinterpret_cast<const __half2*>(&a0), *reinterpret_cast<const __half2*>(&a1))) *
                               mult[32 + t]);
      }
    }
  }
  if (live < kBlockTokens) {   // an open page: its values in fp16
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (is_v ? tid - D : tid) + u * D, l = i & 31, c8 = i >> 5;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float2 f = unpack_half2(x[u][k]);
        if (!is_v) {
          const int t = (c8 / (D / 64)) * 8 + (l >> 2), d = (c8 % (D / 64)) * 64 + (l & 3) * 16 + 2 * k;
          if (t >= live) continue;
          const int slot = (t0 + t) % kTailTokens;
          *reinterpret_cast<uint32_t*>(to.k + (int64_t)slot * D + d) = pack_half2(f.x * mult[t], f.y * mult[t]);
        } else {
          const int b = k >> 1, t = 16 * (c8 / (D / 32)) + 2 * (l & 3) + (b & 1) + 8 * (b >> 1);
          const int d = 32 * (c8 % (D / 32)) + (l >> 2) + 16 * (k & 1);
          if (t >= live) continue;
          const int slot = (t0 + t) % kTailTokens;
          to.v[(int64_t)d * kTailTokens + slot] = __float2half_rn(f.x * mult[32 + t]);
          to.v[(int64_t)(d + 8) * kTailTokens + slot] = __float2half_rn(f.y * mult[32 + t]);
        }
      }
    }
    return;
  }
  char* dst = a.dst.pool + phys_block(a.dst, page) * a.dst.block_bytes + h * a.dst.head_bytes;
  const float2 sc = seal_scale<D, E4M3>(kmax, vmax, red, dst);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = (is_v ? tid - D : tid) + u * D, l = i & 31, c8 = i >> 5;
    float v[4][4];
    uint32_t w[4];
    if (!is_v) {
      const float m = mult[(c8 / (D / 64)) * 8 + (l >> 2)];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float2 f = unpack_half2(x[u][k]);
        v[k >> 1][(k & 1) * 2] = f.x * m;
        v[k >> 1][(k & 1) * 2 + 1] = f.y * m;
      }
    } else {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const float m = mult[32 + 16 * (c8 / (D / 32)) + 2 * (l & 3) + (b & 1) + 8 * (b >> 1)];
        const float2 f0 = unpack_half2(x[u][2 * b]), f1 = unpack_half2(x[u][2 * b + 1]);
        v[0][b] = f0.x * m;
        v[1][b] = f0.y * m;
        v[2][b] = f1.x * m;
        v[3][b] = f1.y * m;
      }
    }
    encode16<E4M3>(v, sc.x, sc.y, w);
    reinterpret_cast<uint4*>(dst + (is_v ? S::kOffV : S::kOffK))[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace lfm3a
