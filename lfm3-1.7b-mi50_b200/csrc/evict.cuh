// Eviction from the 8-bit cache by accumulated attention weight: which keys of each kv head stay (evict_select_kernel)
// and their move into a smaller cache (kv8_compact_kernel).
#pragma once
#include <cooperative_groups.h>

#include "kv8.cuh"

namespace lfm3a {

// Keys of a block's share kept in shared memory; a longer share is read from global memory (L2) on every pass.
constexpr int kEvictCache = 48 * 1024;
struct EvictArgs {
  const float* w;        // [kv_heads][stride]
  int32_t* keep;         // [kv_heads][budget], ascending
  float* w_out;          // [kv_heads][out_stride] weights of the kept keys, or null
  int64_t stride, out_stride;
  int len, sink, recent, budget;
  int cached;            // the blocks' shares fit kEvictCache
};

constexpr int kEvictCluster = 8, kEvictThreads = 1024;

// Weights as unsigned integers of the same order; the zeros are equal and NaN is below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w + 0.f);   // -0 + 0 = +0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One cluster of 8 blocks per kv head: each block owns an eighth of the positions [sink, len - recent), in order. The
// k-th largest weight key is found 8 bits at a time from histograms summed over the cluster's shared memory (every
// block adds up all eight, so all know the same digit); then the blocks write the kept positions in order, starting
// where the counts of the blocks before them end. Of keys equal to the last one kept the first ones stay, so the
// result does not depend on any order of execution.
__global__ __cluster_dims__(kEvictCluster, 1, 1) __launch_bounds__(kEvictThreads) void evict_select_kernel(EvictArgs a) {
  namespace cg = cooperative_groups;
  __shared__ uint32_t hist[2][256];
  __shared__ uint32_t total[256];
  __shared__ uint32_t digit, above;
  __shared__ uint32_t counts[2];       // this block's keys above the threshold, and equal to it
  __shared__ uint32_t warp_sum[32];
  extern __shared__ __align__(1024) uint8_t smem[];
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  pdl_wait();
  pdl_trigger();
  const int rank = (int)cluster.block_rank(), h = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float* w = a.w + h * a.stride;
  int32_t* keep = a.keep + (int64_t)h * a.budget;
  float* w_out = a.w_out ? a.w_out + h * a.out_stride : nullptr;
  const int n = a.len - a.sink - a.recent, k = a.budget - a.sink - a.recent;
  const int i0 = a.sink + (int)((int64_t)n * rank / kEvictCluster);
  const int i1 = a.sink + (int)((int64_t)n * (rank + 1) / kEvictCluster);

  // A thread only ever looks at the keys it put there itself.
  if (a.cached) {
#pragma unroll 8
    for (int i = i0 + tid; i < i1; i += kEvictThreads) keys[i - i0] = weight_key(w[i]);
  }
  auto key_at = [&](int i) { return a.cached ? keys[i - i0] : weight_key(w[i]); };
  uint32_t prefix = 0, mask = 0;      // digits found so far
  int left = k;                       // how many of the keys that match the prefix stay
  if (k > 0 && k < n) {               // the same in every thread of the cluster
    for (int shift = 24, pass = 0; shift >= 0; shift -= 8, ++pass) {
      uint32_t* mine = hist[pass & 1];
      if (tid < 256) mine[tid] = 0;
      __syncthreads();
#pragma unroll 4
      for (int i = i0 + tid; i < i1; i += kEvictThreads) {
        const uint32_t key = key_at(i);
        if ((key & mask) == prefix) atomicAdd(&mine[(key >> shift) & 255u], 1u);
      }
      cluster.sync();
      if (tid < 256) {
        uint32_t sum = 0;
        for (int r = 0; r < kEvictCluster; ++r) sum += cluster.map_shared_rank(mine, r)[tid];
        total[tid] = sum;
      }
      __syncthreads();
      if (warp == 0) {   // the digit at which the count from the top reaches `left`
        uint32_t own[8], sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          own[j] = total[255 - (8 * lane + j)];
          sum += own[j];
        }
        uint32_t incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t u = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += u;
        }
        uint32_t before = incl - sum;
        if (before < (uint32_t)left && incl >= (uint32_t)left) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (before < (uint32_t)left && before + own[j] >= (uint32_t)left) {
              digit = 255 - (8 * lane + j);
              above = before;
            }
            before += own[j];
          }
        }
      }
      __syncthreads();
      prefix |= digit << shift;
      mask |= 255u << shift;
      left -= (int)above;
      __syncthreads();   // digit and above are read
    }
  } else if (k >= n) {   // everything stays: the threshold is below every key
    prefix = 0;
    left = n;
  }
  const bool all = k >= n;

  // Counts of this block's keys above the threshold and equal to it.
  if (tid < 2) counts[tid] = 0;
  __syncthreads();
  uint32_t gt = 0, eq = 0;
  if (k > 0)
#pragma unroll 4
    for (int i = i0 + tid; i < i1; i += kEvictThreads) {
      const uint32_t key = key_at(i);
      gt += all || key > prefix;
      eq += !all && key == prefix;
    }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    gt += __shfl_xor_sync(0xffffffffu, gt, o);
    eq += __shfl_xor_sync(0xffffffffu, eq, o);
  }
  if (lane == 0) {
    atomicAdd(&counts[0], gt);
    atomicAdd(&counts[1], eq);
  }
  cluster.sync();
  uint32_t gt0 = 0, eq0 = 0;   // of the blocks before this one
  for (int r = 0; r < rank; ++r) {
    const uint32_t* c = cluster.map_shared_rank(counts, r);
    gt0 += c[0];
    eq0 += c[1];
  }
  cluster.sync();   // no block leaves while another reads its counts

  if (rank == 0)
    for (int i = tid; i < a.sink; i += kEvictThreads) {
      keep[i] = i;
      if (w_out) w_out[i] = w[i];
    }
  if (rank == kEvictCluster - 1)
    for (int i = tid; i < a.recent; i += kEvictThreads) {
      const int pos = a.len - a.recent + i, at = a.budget - a.recent + i;
      keep[at] = pos;
      if (w_out) w_out[at] = w[pos];
    }
  if (k <= 0) return;
  // In order, 1024 positions at a time: (above, equal) counts of the lanes before as one packed prefix sum.
  for (int base = i0; base < i1; base += kEvictThreads) {
    const int i = base + tid;
    bool is_gt = false, is_eq = false;
    if (i < i1) {
      const uint32_t key = key_at(i);
      is_gt = all || key > prefix;
      is_eq = !all && key == prefix;
    }
    const uint32_t bg = __ballot_sync(0xffffffffu, is_gt), be = __ballot_sync(0xffffffffu, is_eq);
    const uint32_t below = (1u << lane) - 1u;
    uint32_t mine = (uint32_t)__popc(bg & below) | ((uint32_t)__popc(be & below) << 16);
    if (lane == 0) warp_sum[warp] = (uint32_t)__popc(bg) | ((uint32_t)__popc(be) << 16);
    __syncthreads();
    if (warp == 0) {
      uint32_t v = warp_sum[lane];
      const uint32_t own = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      warp_sum[lane] = v - own;
      if (lane == 31) total[0] = v;
    }
    __syncthreads();
    mine += warp_sum[warp];   // at most 1024 of each: the halves do not carry
    const uint32_t my_gt = gt0 + (mine & 0xffffu), my_eq = eq0 + (mine >> 16);
    if (is_gt || (is_eq && my_eq < (uint32_t)left)) {
      const int at = a.sink + (int)(my_gt + min(my_eq, (uint32_t)left));
      keep[at] = i;
      if (w_out) w_out[at] = w[i];
    }
    const uint32_t t = total[0];
    gt0 += t & 0xffffu;
    eq0 += t >> 16;
    __syncthreads();   // warp_sum and total are free
  }
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
// A token's K is one contiguous run of its section, its V one byte in each word of D / 4 chunks; a thread has all its
// loads in flight at once (taken one after the other, their latency was the whole time).
template <int D, bool E4M3>
__global__ __launch_bounds__(kSealThreads) void kv8_compact_kernel(Kv8CompactArgs a) {
  using S = Q8Section<D>;
  constexpr int RS = kSealRow<D>, KI = 2 * D / kSealThreads > 0 ? 2 * D / kSealThreads : 1, VI = 8 * D / kSealThreads;
  __shared__ __align__(16) float x[2 * 32 * RS];
  __shared__ __align__(16) uint8_t codes[32 * D];
  __shared__ float red[16];
  __shared__ const char* sec[32];
  __shared__ int pos[32];
  __shared__ float2 scales[32];
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, page = blockIdx.x, h = blockIdx.y, t0 = page * kBlockTokens;
  const int live = min(kBlockTokens, a.budget - t0);
  if (tid < live) {
    const int p = min(max(a.keep[(int64_t)h * a.budget + t0 + tid], 0), a.len - 1);
    pos[tid] = p;
    const char* s = nullptr;
    if (p < a.sealed) {
      s = a.src.pool + phys_block(a.src, p / kBlockTokens) * a.src.block_bytes + h * a.src.head_bytes;
      const float2 f = *reinterpret_cast<const float2*>(s);
      scales[tid] = make_float2(f.x * kCodeUnit<E4M3>, f.y * kCodeUnit<E4M3>);
    }
    sec[tid] = s;
  }
  __syncthreads();
  const TailView from = tail_of(a.src_tail, a.src.kv_heads, h, D);
  float kmax = 0.f, vmax = 0.f;
  uint4 kr[KI], vr[VI];   // 16 dims of one token's K; 4 dims of one token's V (a byte of each word)
#pragma unroll
  for (int u = 0; u < KI; ++u) {
    const int i = tid + u * kSealThreads, t = i / (D / 16), d0 = (i % (D / 16)) * 16;
    kr[u] = make_uint4(0, 0, 0, 0);
    if (i < 2 * D && t < live && sec[t])
      kr[u] = *reinterpret_cast<const uint4*>(sec[t] + S::kOffK + S::k_chunk(pos[t] % kBlockTokens, d0) * 16);
  }
#pragma unroll
  for (int u = 0; u < VI; ++u) {
    const int i = tid + u * kSealThreads, t = i / (D / 4), k = i % (D / 4);   // chunk (dim pair of tiles k / 8, g = k % 8)
    vr[u] = make_uint4(0, 0, 0, 0);
    if (t < live && sec[t])
      vr[u] = *reinterpret_cast<const uint4*>(sec[t] + S::kOffV + S::v_index(pos[t] % kBlockTokens & ~9, 32 * (k >> 3) + (k & 7)));
  }
#pragma unroll
  for (int u = 0; u < KI; ++u) {
    const int i = tid + u * kSealThreads, t = i / (D / 16), d0 = (i % (D / 16)) * 16;
    if (i >= 2 * D || t >= live) continue;
    float* row = x + t * RS + d0;
    if (sec[t]) {
      const float ks = scales[t].x;
      const uint32_t w[4] = {kr[u].x, kr[u].y, kr[u].z, kr[u].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 p = unpack_half2(decode_pair<E4M3, false>(w[k])), q = unpack_half2(decode_pair<E4M3, true>(w[k]));
        const float4 f = make_float4(p.x * ks, p.y * ks, q.x * ks, q.y * ks);
        *reinterpret_cast<float4*>(row + 4 * k) = f;
        kmax = fmaxf(kmax, fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w))));
      }
    } else {
      const __half* src = from.k + (int64_t)(pos[t] % kTailTokens) * D + d0;
      kmax = fmaxf(kmax, stage_row8(src, true, row));
      kmax = fmaxf(kmax, stage_row8(src + 8, true, row + 8));
    }
  }
#pragma unroll
  for (int u = 0; u < VI; ++u) {
    const int i = tid + u * kSealThreads, t = i / (D / 4), k = i % (D / 4), d0 = 32 * (k >> 3) + (k & 7);
    if (t >= live) continue;
    const int p = pos[t], byte = (p >> 3 & 1) * 2 + (p & 1);
    const uint32_t w[4] = {vr[u].x, vr[u].y, vr[u].z, vr[u].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = d0 + 8 * e;
      float f;
      if (sec[t]) f = unpack_half2(decode_pair<E4M3, false>(w[e] >> (8 * byte) & 0xffu)).x * scales[t].y;
      else f = __half2float(from.v[(int64_t)d * kTailTokens + p % kTailTokens]);
      x[(32 + t) * RS + d] = f;
      vmax = fmaxf(vmax, fabsf(f));
    }
  }
  if (live == kBlockTokens) {
    seal_page<D, E4M3>(x, kmax, vmax, red, codes, a.dst.pool + phys_block(a.dst, page) * a.dst.block_bytes + h * a.dst.head_bytes);
    return;
  }
  __syncthreads();
  const TailView to = tail_of(a.dst_tail, a.dst.kv_heads, h, D);
  for (int i = tid; i < live * D; i += kSealThreads) {
    const int t = i / D, d = i % D, slot = (t0 + t) % kTailTokens;
    to.k[(int64_t)slot * D + d] = __float2half_rn(x[t * RS + d]);
    to.v[(int64_t)d * kTailTokens + slot] = __float2half_rn(x[(32 + t) * RS + d]);
  }
}

}  // namespace lfm3a
