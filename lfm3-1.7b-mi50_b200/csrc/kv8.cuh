// The 8-bit KV cache with a scale per block of 32 tokens and kv head (LFM3A_MODE_I8BLK: int8, LFM3A_MODE_E4M3BLK: fp8
// e4m3): append and sealing, reading back, attention, prefill staging and per-key attention weights.
//
// A page is one block. Pages that are complete and committed are sealed: x is held as q = round8(x / s), with
// s = absmax / 127 (448 for e4m3; 1 for a block of zeros) over the page's 32 x D values of the head, K and V each; an
// int8 is stored as the byte q + 128.
// The last tokens (an incomplete page, drafts that may be rolled back) stay in fp16 in a ring of 128 tokens per layer,
// the tail, so a sealed page depends on committed tokens alone and a rollback needs no device work.
//
// Section of one (page, kv head), 32 + 64 D bytes: f32 K scale, f32 V scale, 4 zero bytes, f32 V factor of the attention
// kernels' P (the V scale, but 2^-40 for a block of zeros), 16 zero bytes, K (32 D bytes), V (32 D).
// K and V lie in the order in which the lanes of a warp (g = lane / 4, c = lane % 4) take them as the A operands of
// mma.m16n8k16: S^T = K Q^T over 16 keys x 8 query rows, and O^T = V^T P over 16 dims x 8 rows. A dot over dims does
// not care which dim sits at which k, so a lane takes 16 contiguous dims of a key in one 16-byte load:
//   K byte (key, dim): chunk ((key / 16 * 2 + key / 8 % 2) * (D / 64) + dim / 64) * 32 + (key % 8) * 4 + dim / 16 % 4,
//                      byte dim % 16
//   V byte (key, dim): chunk (key / 16 * (D / 32) + dim / 32) * 32 + (dim % 8) * 4 + key % 8 / 2,
//                      byte dim / 16 % 2 * 8 + dim / 8 % 2 * 4 + key / 8 % 2 * 2 + key % 2
// so every shared-memory load of a fragment is 32 consecutive 16-byte chunks, without bank conflicts.
#pragma once
#include <cooperative_groups.h>

#include "common.cuh"
#include "i8rec.cuh"
#include "kv.cuh"
#include "verify.cuh"

namespace lfm3a {

namespace cg = cooperative_groups;

constexpr int kTailTokens = 128;   // tokens of the fp16 tail ring (slot = position mod 128)
// V factor of a block of zeros: any serves, its codes being zeros, but a factor above its neighbours' scales would raise
// the running maximum and push their P out of fp16 (with 1 beside V of 1e-4, e4m3, outputs are off by 0.008 of the RMS).
constexpr float kZeroFactor = 0x1p-40f;
constexpr int kFactorWord = 3;     // its place in a section

template <int D>
struct Q8Section {
  static constexpr int kHeader = 32;
  static constexpr int kOffK = kHeader, kOffV = kHeader + 32 * D, kBytes = kHeader + 64 * D;
  __host__ __device__ __forceinline__ static constexpr int k_chunk(int key, int dim) {
    return (((key >> 4) * 2 + ((key >> 3) & 1)) * (D / 64) + (dim >> 6)) * 32 + (key & 7) * 4 + ((dim >> 4) & 3);
  }
  __host__ __device__ __forceinline__ static constexpr int v_index(int key, int dim) {
    return (((key >> 4) * (D / 32) + (dim >> 5)) * 32 + (dim & 7) * 4 + ((key & 7) >> 1)) * 16 + ((dim >> 4) & 1) * 8 +
           ((dim >> 3) & 1) * 4 + ((key >> 3) & 1) * 2 + (key & 1);
  }
};

// The tail: K [kv_heads][128 slots][D], then V transposed, [kv_heads][D][128 slots] (pairs of keys in one word).
struct TailView {
  __half* k;
  __half* v;
};
__host__ __device__ __forceinline__ TailView tail_of(__half* tail, int kv_heads, int h, int D) {
  TailView t;
  t.k = tail + (int64_t)h * kTailTokens * D;
  t.v = tail + (int64_t)(kv_heads + h) * kTailTokens * D;
  return t;
}

// fp16 values of the cache are finite: NaN becomes 0, an infinity the largest finite value of its sign.
__device__ __forceinline__ float finite_f16(float x) { return x != x ? 0.f : fminf(fmaxf(x, -65504.f), 65504.f); }

// Four words of 8-bit codes, byte b of word k being the code of the fp32 quotient v[k][b] / scale, to nearest even (inv:
// the rounded reciprocal of scale; no value is beyond 127 or 448 scales). v * inv is within 2^-22 of the quotient,
// relatively, so it decides a code unless a rounding boundary lies that near; if one does for any of the 16, the
// divisions themselves decide all of them. (Dividing every value took half of the append kernel's time, a branch per
// value another quarter.)
template <bool E4M3>
__device__ __forceinline__ void encode16(const float (&v)[4][4], float scale, float inv, uint32_t (&w)[4]) {
  if (E4M3) {   // saturating at 448
    auto pair = [](float lo, float hi) {
      uint16_t r;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
      return (uint32_t)r;
    };
    uint32_t doubt = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t r[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float y0 = v[k][2 * b] * inv, y1 = v[k][2 * b + 1] * inv;
        r[b] = pair(y0 * (1.f + 0x1p-21f), y1 * (1.f + 0x1p-21f));
        doubt |= r[b] ^ pair(y0 * (1.f - 0x1p-21f), y1 * (1.f - 0x1p-21f));
      }
      w[k] = __byte_perm(r[0], r[1], 0x5410);
    }
    if (doubt) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w[k] = __byte_perm(pair(__fdiv_rn(v[k][0], scale), __fdiv_rn(v[k][1], scale)),
                           pair(__fdiv_rn(v[k][2], scale), __fdiv_rn(v[k][3], scale)), 0x5410);
    }
    return;
  }
  constexpr float kMagic = 12582912.f + 128.f;   // 1.5 * 2^23: adding it rounds to an integer; the code is stored plus 128
  float t[4][4], worst = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      t[k][b] = fmaf(v[k][b], inv, kMagic);
      worst = fmaxf(worst, fabsf(fmaf(v[k][b], inv, kMagic - t[k][b])));
    }
  if (worst > 0.49998f) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int b = 0; b < 4; ++b) t[k][b] = __fdiv_rn(v[k][b], scale) + kMagic;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    w[k] = __byte_perm(__byte_perm(__float_as_uint(t[k][0]), __float_as_uint(t[k][1]), 0x0040),
                       __byte_perm(__float_as_uint(t[k][2]), __float_as_uint(t[k][3]), 0x0040), 0x5410);
}

// Bytes 0, 1 (or with HI 2, 3) of a word of codes as an fp16 pair, exactly. decode_raw is one instruction: the byte v + 128
// of an int8 is, as the bits of a subnormal fp16, (v + 128) 2^-24; the unit goes into K's scale (kCodeUnit), and the
// scores start from minus 128 times the row's sum of q. decode_pair gives the values: V's sums run over thousands of keys,
// and with a bias of 128 in them the tensor cores' fp32 accumulation cost 8 times the error (0.0017 of the RMS over 131072).
template <bool E4M3>
constexpr float kCodeUnit = E4M3 ? 1.f : 0x1p24f;
template <bool E4M3>
constexpr float kCodeBias = E4M3 ? 0.f : 128.f * 0x1p-24f;
template <bool E4M3, bool HI>
__device__ __forceinline__ uint32_t decode_raw(uint32_t w) {
  if (E4M3) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(HI ? w >> 16 : w)));
    return h;
  }
  return __byte_perm(w, 0u, HI ? 0x4342 : 0x4140);
}
template <bool E4M3, bool HI>
__device__ __forceinline__ uint32_t decode_pair(uint32_t w) {
  if (E4M3) return decode_raw<E4M3, HI>(w);
  const uint32_t h = __byte_perm(w, 0x64u, HI ? 0x4342 : 0x4140);   // 0x64NN: 1024 + NN
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h), __floats2half2_rn(1152.f, 1152.f));
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// ---------------------------------------------------------------- append and sealing
// A page and kv head is sealed by 2 D threads: the first half of them makes K's codes, the other V's, 16 at a time, two
// times each. Each gives the largest magnitude of the K and of the V values it has seen and gets the scale of its half
// and the rounded reciprocal; the header (both scales, the V factor, zeros) is written. The barrier inside also publishes
// shared memory written before.
template <int D>
constexpr int kSealThreads = 2 * D;
template <int D, bool E4M3>
__device__ __forceinline__ float2 seal_scale(float kmax, float vmax, float* red, char* sec) {
  constexpr int W = kSealThreads<D> / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    kmax = fmaxf(kmax, __shfl_xor_sync(0xffffffffu, kmax, o));
    vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
  }
  if (lane == 0) {
    red[warp] = kmax;
    red[W + warp] = vmax;
  }
  __syncthreads();
  const bool is_v = tid >= D;
  const float4* r = reinterpret_cast<const float4*>(red + (is_v ? W : 0));
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < W / 4; ++i) amax = fmaxf(amax, fmaxf(fmaxf(r[i].x, r[i].y), fmaxf(r[i].z, r[i].w)));
  const float scale = amax > 0.f ? __fdiv_rn(amax, E4M3 ? 448.f : 127.f) : 1.f;
  if (lane < 4 && (warp == 0 || warp == W / 2)) {
    const int word = 2 * lane + is_v;
    reinterpret_cast<float*>(sec)[word] = lane == 0 ? scale : word == kFactorWord ? (amax > 0.f ? scale : kZeroFactor) : 0.f;
  }
  return make_float2(scale, __fdiv_rn(1.f, scale));
}

template <int D>
constexpr int kSealRow = D + 8;   // halves of a staged row; 16-byte aligned rows
__device__ __forceinline__ void unpack4(uint2 h, float (&f)[4]) {
  const float2 a = unpack_half2(h.x), b = unpack_half2(h.y);
  f[0] = a.x;
  f[1] = a.y;
  f[2] = b.x;
  f[3] = b.y;
}
// Seals fp16 rows staged in shared memory (x [2][32][kSealRow]: K, then V). A thread makes a whole 16-byte chunk of K at a
// time, or 4 dims x 4 keys of V: four words, of which 16 lanes' fill 64 bytes.
template <int D, bool E4M3>
__device__ __forceinline__ void seal_page(const __half* x, float kmax, float vmax, float* red, char* sec) {
  using S = Q8Section<D>;
  constexpr int RS = kSealRow<D>;
  const int tid = threadIdx.x;
  const float2 sc = seal_scale<D, E4M3>(kmax, vmax, red, sec);
  uint32_t w[4];
  float v[4][4];
  if (tid < D) {
    uint4* K = reinterpret_cast<uint4*>(sec + S::kOffK);
#pragma unroll
    for (int i = tid; i < 2 * D; i += D) {   // 16 dims of one key
      const int l = i & 31, a = i >> 5;
      const int key = (a / (D / 64)) * 8 + (l >> 2), dim0 = (a % (D / 64)) * 64 + (l & 3) * 16;
      const uint4* src = reinterpret_cast<const uint4*>(x + key * RS + dim0);
      const uint4 a0 = src[0], a1 = src[1];
      unpack4(make_uint2(a0.x, a0.y), v[0]);
      unpack4(make_uint2(a0.z, a0.w), v[1]);
      unpack4(make_uint2(a1.x, a1.y), v[2]);
      unpack4(make_uint2(a1.z, a1.w), v[3]);
      encode16<E4M3>(v, sc.x, sc.y, w);
      K[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
    uint8_t* V = reinterpret_cast<uint8_t*>(sec + S::kOffV);
#pragma unroll
    for (int i = tid - D; i < 2 * D; i += D) {   // dims dim0 .. + 3 of 4 keys
      const int c = i & 3, wi = (i >> 2) & 3, gh = (i >> 4) & 1, dtp = (i >> 5) % (D / 32), mt = (i >> 5) / (D / 32);
      const int key0 = 16 * mt + 2 * c, dim0 = 32 * dtp + 16 * (wi >> 1) + 8 * (wi & 1) + 4 * gh;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        float f[4];
        unpack4(*reinterpret_cast<const uint2*>(x + (32 + key0 + (b & 1) + 8 * (b >> 1)) * RS + dim0), f);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e][b] = f[e];
      }
      encode16<E4M3>(v, sc.x, sc.y, w);
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<uint32_t*>(V + S::v_index(key0, dim0 + e)) = w[e];
    }
  }
}

// 8 halves at p (16-byte aligned when vec).
__device__ __forceinline__ uint4 load_row8(const __half* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __halves2half2(p[2 * i], p[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Largest magnitude of 8 halves, NaN if one is.
__device__ __forceinline__ __half2 max_abs8(uint4 v, __half2 m) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = w[i] & 0x7fff7fffu;
    m = __hmax2_nan(m, *reinterpret_cast<const __half2*>(&a));
  }
  return m;
}
__device__ __forceinline__ float max_of(__half2 m) {
  const __half h = __hmax_nan(__low2half(m), __high2half(m));
  return __half2float(h);
}
// Makes 8 halves finite in place; returns their largest magnitude.
__device__ __forceinline__ float make_finite8(__half* p) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = finite_f16(__half2float(p[i]));
    p[i] = __float2half_rn(f);
    m = fmaxf(m, fabsf(f));
  }
  return m;
}

struct Kv8AppendArgs {
  AppendArgs a;      // pool geometry, new rows, RoPE table, k-norm, pos0, n
  __half* tail;
  int page0;         // first page of the launch
  int seal_page_end; // pages below are sealed, the others go to the tail
  int vec;           // rows of k and v start 16-byte aligned
};

// One block per (page, kv head): the page's tokens below pos0 come from the tail, the others from the new rows (8 values
// a load; K through the fp16 k-norm and RoPE that lfm3a_kv_append applies). Bound by memory for prompt chunks, by the
// latency of one round of loads for drafts. 131072 tokens at 8 heads of 64 (int8) take 92 us (4.4 TB/s), instructions
// and memory about even; 7680 at 4 of 128 (e4m3) 9 us.
template <int D, bool E4M3>
__global__ __launch_bounds__(kSealThreads<D>) void kv8_append_kernel(Kv8AppendArgs args) {
  constexpr int J = D / 64, HALF = D / 2, RS = kSealRow<D>, R8 = D / 8;
  __shared__ __align__(16) __half x[2 * 32 * RS];
  __shared__ __align__(16) float red[16];
  pdl_wait();
  pdl_trigger();
  const AppendArgs& a = args.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int page = args.page0 + blockIdx.x, h = blockIdx.y, t0 = page * kBlockTokens;
  const int lo = max(t0, a.pos0), end = min(t0 + kBlockTokens, a.pos0 + a.n);   // new tokens
  const bool sealing = page < args.seal_page_end, vec = args.vec != 0, plain = !a.knorm && !a.rope;
  if (!sealing && lo >= end) return;
  const TailView tail = tail_of(args.tail, a.g.kv_heads, h, D);
  float kmax = 0.f, vmax = 0.f;
  {
    constexpr int U = kBlockTokens * R8 / kSealThreads<D>;   // 16-byte pieces of K and of V per thread
    uint4 kr[U], vr[U];
    const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = tid + u * kSealThreads<D>, t = t0 + i / R8;
      const bool live = t >= lo && t < end;
      const int64_t at = (int64_t)(t - a.pos0) * a.stride + h * D + (i % R8) * 8;
      kr[u] = live && plain ? load_row8(a.k + at, vec) : zero;
      vr[u] = live ? load_row8(a.v + at, vec) : zero;
    }
    __half2 km = __float2half2_rn(0.f), vm = km;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = tid + u * kSealThreads<D>, r = i / R8, d = (i % R8) * 8;
      if (t0 + r >= lo && t0 + r < end) {
        if (plain) *reinterpret_cast<uint4*>(x + r * RS + d) = kr[u];
        *reinterpret_cast<uint4*>(x + (32 + r) * RS + d) = vr[u];
      }
      km = max_abs8(kr[u], km);
      vm = max_abs8(vr[u], vm);
    }
    kmax = max_of(km);
    vmax = max_of(vm);
    if (!(kmax <= 65504.f) || !(vmax <= 65504.f)) {   // an infinity or NaN among this thread's values
      kmax = vmax = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = tid + u * kSealThreads<D>, r = i / R8, d = (i % R8) * 8;
        if (t0 + r < lo || t0 + r >= end) continue;
        if (plain) kmax = fmaxf(kmax, make_finite8(x + r * RS + d));
        vmax = fmaxf(vmax, make_finite8(x + (32 + r) * RS + d));
      }
    }
  }
  if (!plain) {
#pragma unroll 4
    for (int t = lo + warp; t < end; t += kSealThreads<D> / 32) {
      float ra[J], rb[J];
      norm_rope_pairs<D>(a, a.k + (int64_t)(t - a.pos0) * a.stride + h * D, t, lane, ra, rb);
      __half* row = x + (t - t0) * RS;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float k0 = finite_f16(ra[j]), k1 = finite_f16(rb[j]);
        row[lane + 32 * j] = __float2half_rn(k0);
        row[lane + 32 * j + HALF] = __float2half_rn(k1);
        kmax = fmaxf(kmax, fmaxf(fabsf(k0), fabsf(k1)));
      }
    }
  }
  if (!sealing) {
    __syncthreads();
    for (int i = tid; i < (end - lo) * D; i += kSealThreads<D>) {
      const int t = lo + i / D, d = i % D, slot = t % kTailTokens;
      tail.k[(int64_t)slot * D + d] = x[(t - t0) * RS + d];
      tail.v[(int64_t)d * kTailTokens + slot] = x[(32 + t - t0) * RS + d];
    }
    return;
  }
  if (lo > t0) {   // tokens that wait in the tail (finite already)
    const int old = min(lo, t0 + kBlockTokens) - t0, slot0 = t0 % kTailTokens;
    __half2 km = __float2half2_rn(0.f);
    for (int i = tid; i < old * R8; i += kSealThreads<D>) {
      const int r = i / R8, d = (i % R8) * 8;
      const uint4 v = *reinterpret_cast<const uint4*>(tail.k + (int64_t)(slot0 + r) * D + d);
      *reinterpret_cast<uint4*>(x + r * RS + d) = v;
      km = max_abs8(v, km);
    }
    kmax = fmaxf(kmax, max_of(km));
    for (int i = tid; i < D * 4; i += kSealThreads<D>) {   // 8 tokens of one dim
      const int d = i >> 2, r0 = (i & 3) * 8;
      if (r0 >= old) continue;
      const uint4 v = *reinterpret_cast<const uint4*>(tail.v + (int64_t)d * kTailTokens + slot0 + r0);
      const __half* f = reinterpret_cast<const __half*>(&v);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (r0 + e < old) {
          x[(32 + r0 + e) * RS + d] = f[e];
          vmax = fmaxf(vmax, fabsf(__half2float(f[e])));
        }
    }
  }
  seal_page<D, E4M3>(x, kmax, vmax, red, a.g.pool + phys_block(a.g, page) * a.g.block_bytes + h * a.g.head_bytes);
}

// ---------------------------------------------------------------- reading back
struct Kv8ReadArgs {
  KvGeom g;
  __half* tail;
  __half* k;       // [n][kv_heads][D]
  __half* v;
  int pos0, n, sealed;
};

// One block per (page, kv head): the values the cache stands for, rounded to fp16; 16-byte stores of 8 dims of a token.
// Bound by memory: 32768 tokens at 8 heads of 64 take 16.8 us (6.0 TB/s).
template <int D, bool E4M3>
__global__ __launch_bounds__(128) void kv8_read_kernel(Kv8ReadArgs a) {
  using S = Q8Section<D>;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, page = a.pos0 / kBlockTokens + blockIdx.x, h = blockIdx.y, t0 = page * kBlockTokens;
  const int lo = max(a.pos0, t0), hi = min(a.pos0 + a.n, t0 + kBlockTokens);
  const int64_t row = (int64_t)a.g.kv_heads * D;
  __half* const k_out = a.k + h * D;
  __half* const v_out = a.v + h * D;
  if (t0 < a.sealed) {
    const char* sec = a.g.pool + phys_block(a.g, page) * a.g.block_bytes + h * a.g.head_bytes;
    const float ks = reinterpret_cast<const float*>(sec)[0];
    const float vs = reinterpret_cast<const float*>(sec)[1];
    const uint4* K = reinterpret_cast<const uint4*>(sec + S::kOffK);
    const uint32_t* V = reinterpret_cast<const uint32_t*>(sec + S::kOffV);
#pragma unroll
    for (int i = tid; i < 2 * D; i += 128) {   // 16 dims of one key
      const int l = i & 31, s = i >> 5;
      const int t = t0 + (s / (D / 64)) * 8 + (l >> 2), d = (s % (D / 64)) * 64 + (l & 3) * 16;
      const uint4 r = K[i];
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
      uint32_t o[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 p = unpack_half2(decode_pair<E4M3, false>(w[k])), q = unpack_half2(decode_pair<E4M3, true>(w[k]));
        o[2 * k] = pack_half2(p.x * ks, p.y * ks);
        o[2 * k + 1] = pack_half2(q.x * ks, q.y * ks);
      }
      if (t < lo || t >= hi) continue;
      uint4* dst = reinterpret_cast<uint4*>(k_out + (t - a.pos0) * row + d);
      dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
      dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
#pragma unroll
    for (int i = tid; i < D; i += 128) {   // 8 dims (one word each) of keys key0, + 1, + 8, + 9
      const int c = i & 3, wi = (i >> 2) & 3, dtp = (i >> 4) % (D / 32), mt = (i >> 4) / (D / 32);
      const int key0 = 16 * mt + 2 * c, d = 32 * dtp + 16 * (wi >> 1) + 8 * (wi & 1);
      uint32_t w[8];
#pragma unroll
      for (int g = 0; g < 8; ++g) w[g] = V[S::v_index(key0, d + g) / 4];
      float f[4][8];
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        const float2 p = unpack_half2(decode_pair<E4M3, false>(w[g])), q = unpack_half2(decode_pair<E4M3, true>(w[g]));
        f[0][g] = p.x * vs;
        f[1][g] = p.y * vs;
        f[2][g] = q.x * vs;
        f[3][g] = q.y * vs;
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int t = t0 + key0 + (b & 1) + 8 * (b >> 1);
        if (t < lo || t >= hi) continue;
        *reinterpret_cast<uint4*>(v_out + (t - a.pos0) * row + d) =
            make_uint4(pack_half2(f[b][0], f[b][1]), pack_half2(f[b][2], f[b][3]), pack_half2(f[b][4], f[b][5]),
                       pack_half2(f[b][6], f[b][7]));
      }
    }
  } else {
    const TailView tail = tail_of(a.tail, a.g.kv_heads, h, D);
    const int slot0 = t0 % kTailTokens;
    constexpr int U = D / 32;   // 8 values of K and of V per thread and round, all loads first
    uint4 kr[U], vr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = tid + 128 * u;
      kr[u] = *reinterpret_cast<const uint4*>(tail.k + (int64_t)(slot0 + i / (D / 8)) * D + (i % (D / 8)) * 8);
      vr[u] = *reinterpret_cast<const uint4*>(tail.v + (int64_t)(i % D) * kTailTokens + slot0 + (i / D) * 8);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = tid + 128 * u, t = t0 + i / (D / 8);
      if (t >= lo && t < hi) *reinterpret_cast<uint4*>(k_out + (t - a.pos0) * row + (i % (D / 8)) * 8) = kr[u];
      const __half* v = reinterpret_cast<const __half*>(&vr[u]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int tv = t0 + (i / D) * 8 + e;
        if (tv >= lo && tv < hi) v_out[(tv - a.pos0) * row + i % D] = v[e];
      }
    }
  }
}

// ---------------------------------------------------------------- attention
struct Kv8AttnArgs {
  KvGeom g;
  __half* tail;
  const __half* q;      // row (t, qh) at q + t * q_stride + qh * D
  const __half* gate;   // [m][q_heads] logits, or null
  __half* out;          // [m][q_heads][D] (one split)
  float* lse;           // [m][q_heads] natural-log sum of exponentials, or null
  float* part;          // [m * q_heads][splits][D + 2] (several splits)
  int64_t q_stride;
  int m, group, q_heads, ctx_len, window, sealed, splits;
  int p_begin, p_total; // pages of [start, ctx_len + m)
  float qk_scale;       // (1 / sqrt(D)) log2(e)
};

// The query rows of one kv head as B operands (r = t * group + j): chunk ((n-tile * D / 64 + e) * 2 + s) * 32 + lane
// holds dims 64 e + 16 c + 8 s .. + 7 of row 8 n-tile + g: b0, b1 of k-steps 2 s and 2 s + 1. Rows past m * group are 0.
template <int D>
__device__ __forceinline__ void stage_q(const __half* q, int64_t q_stride, int rows, int group, int h, int row0, int ntiles,
                                        uint4* sq, int tid, int threads) {
  for (int i = tid; i < ntiles * D; i += threads) {
    const int l = i & 31, k = i >> 5, s = k & 1, e = (k >> 1) % (D / 64), nt = (k >> 1) / (D / 64);
    const int r = row0 + 8 * nt + (l >> 2);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < rows) {
      const int t = r / group, j = r - t * group;
      v = *reinterpret_cast<const uint4*>(q + t * q_stride + (int64_t)(h * group + j) * D + 64 * e + 16 * (l & 3) + 8 * s);
    }
    sq[i] = v;
  }
}

// Whether every row sees every key of the page (rows at ctx_len .. ctx_len + m - 1).
__device__ __forceinline__ bool page_open(int page, int ctx_len, int m, int window) {
  return page * kBlockTokens + kBlockTokens - 1 <= ctx_len &&
         (window == 0 || page * kBlockTokens > ctx_len + m - 1 - window);
}
__device__ __forceinline__ bool sees(int pos, int key, int window) {
  return key <= pos && (window == 0 || key > pos - window);
}

template <int D, int NT>
struct Kv8Attn {
  // Two blocks of 8 warps per SM at head_dim 64 (128 registers), one of 12 at 128 (168).
  static constexpr int kWarps = D == 64 ? 8 : 12, kThreads = 32 * kWarps, kStages = D == 64 ? 3 : 2;
  static constexpr int kStageBytes = Q8Section<D>::kBytes;                 // a multiple of 32
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kOStride = D + 4;                                   // floats, 4 mod 32 banks
  static constexpr int kMerge = kWarps * 8 * NT * (kOStride + 2) * 4;      // over the ring once it is drained
  static constexpr int kFinal = kMerge + 8 * NT * (D + 2) * 4;             // and a split's rows after them
  static constexpr int kOffQ = kRing > kFinal ? kRing : kFinal;
  static constexpr int kOffBias = kOffQ + 8 * NT * D * 2;                  // per row: - kCodeBias times the sum of q
  static constexpr int kOffBar = kOffBias + 8 * NT * 4;
  static constexpr int kSmem = kOffBar + kWarps * kStages * 8;
  static constexpr int kBlocksPerSm = D == 64 ? 2 : 1;
};

// Fragments of a tail page straight from the ring in global memory (fp16, L2-resident).
template <int D>
__device__ __forceinline__ void tail_k_frag(const TailView& t, int key0, int e, int g, int c, uint2 (&kA)[4],
                                            uint2 (&kB)[4]) {
  const uint4* a = reinterpret_cast<const uint4*>(t.k + (int64_t)((key0 + g) % kTailTokens) * D + 64 * e + 16 * c);
  const uint4* b = reinterpret_cast<const uint4*>(t.k + (int64_t)((key0 + g + 8) % kTailTokens) * D + 64 * e + 16 * c);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 x = a[i], y = b[i];
    kA[2 * i] = make_uint2(x.x, x.y);
    kA[2 * i + 1] = make_uint2(x.z, x.w);
    kB[2 * i] = make_uint2(y.x, y.y);
    kB[2 * i + 1] = make_uint2(y.z, y.w);
  }
}
// The pair of keys key, key + 1 (key even) at one dim, 0 past the sequence's end: a stale slot may hold anything.
__device__ __forceinline__ uint32_t tail_v_pair(const TailView& t, int key, int dim, int kv_end) {
  uint32_t w = *reinterpret_cast<const uint32_t*>(t.v + (int64_t)dim * kTailTokens + key % kTailTokens);
  if (key + 1 >= kv_end) w &= key >= kv_end ? 0u : 0xffffu;
  return w;
}

// -kCodeBias times the sum of each query row's values, a row by D / 8 lanes (order fixed). The loads of several rows go out
// together: one row after the other they took 5 us of the weights of 128 rows.
template <int D>
__device__ __forceinline__ void stage_bias(const __half* q, int64_t q_stride, int rows, int group, int h, int row0, int count,
                                           float bias, float* dst, int warp, int warps, int lane) {
  constexpr int R = D / 8, P = 32 / R, U = 4;
  for (int i0 = warp * P + lane / R; i0 - lane / R < count; i0 += U * warps * P) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * warps * P, r = row0 + i;
      v[u] = make_uint4(0, 0, 0, 0);
      if (i < count && r < rows) {
        const int t = r / group, j = r - t * group;
        v[u] = reinterpret_cast<const uint4*>(q + t * q_stride + (int64_t)(h * group + j) * D)[lane % R];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * warps * P;
      const float2 a = fadd2(unpack_half2(v[u].x), unpack_half2(v[u].y)), b = fadd2(unpack_half2(v[u].z), unpack_half2(v[u].w));
      float sum = (a.x + a.y) + (b.x + b.y);
#pragma unroll
      for (int o = R / 2; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane % R == 0 && i < count) dst[i] = -bias * sum;
    }
  }
}

// d = a x b + (c0, c1, c0, c1).
__device__ __forceinline__ void mma_f16_16816_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float2 c) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y));
}

// S^T of the HB 16-key halves of a sealed page and 8 NT query rows, by a warp: s[b][n] is an accumulator of keys
// g, g + 8 (rows) and query rows 2 c, 2 c + 1 (columns). The accumulators start from the bias' share.
template <int D, int NT, int HB, bool E4M3>
struct Kv8Scores {
  const uint8_t* k;      // the page's K codes
  const uint4* sq;
  const float* sbias;
  int lane;
  // The same scores, to be made anew: nothing of an earlier pass is kept in registers for it.
  __device__ __forceinline__ Kv8Scores again() const {
    Kv8Scores q = *this;
    asm volatile("" : "+l"(q.k), "+l"(q.sq), "+l"(q.sbias));
    return q;
  }
  __device__ __forceinline__ void operator()(float (&s)[HB][NT][4]) const {
    constexpr int NE = D / 64;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      uint32_t wa[HB][4], wb[HB][4];
#pragma unroll
      for (int b = 0; b < HB; ++b) {
        const uint4* k4 = reinterpret_cast<const uint4*>(k) + (2 * b * NE + e) * 32 + lane;
        const uint4 ra = k4[0], rb = k4[NE * 32];
        wa[b][0] = ra.x;
        wa[b][1] = ra.y;
        wa[b][2] = ra.z;
        wa[b][3] = ra.w;
        wb[b][0] = rb.x;
        wb[b][1] = rb.y;
        wb[b][2] = rb.z;
        wb[b][3] = rb.w;
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        uint32_t f[HB][2][4];
#pragma unroll
        for (int b = 0; b < HB; ++b)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            f[b][u][0] = decode_raw<E4M3, false>(wa[b][2 * s2 + u]);
            f[b][u][1] = decode_raw<E4M3, false>(wb[b][2 * s2 + u]);
            f[b][u][2] = decode_raw<E4M3, true>(wa[b][2 * s2 + u]);
            f[b][u][3] = decode_raw<E4M3, true>(wb[b][2 * s2 + u]);
          }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 qv = sq[((n * NE + e) * 2 + s2) * 32 + lane];
#pragma unroll
          for (int b = 0; b < HB; ++b) {
            if (e == 0 && s2 == 0) {
              float2 start = make_float2(0.f, 0.f);
              if (!E4M3) start = *reinterpret_cast<const float2*>(sbias + 8 * n + 2 * (lane & 3));
              mma_f16_16816_from(s[b][n], f[b][0], qv.x, qv.y, start);
            } else {
              mma_f16_16816(s[b][n], f[b][0], qv.x, qv.y);
            }
            mma_f16_16816(s[b][n], f[b][1], qv.z, qv.w);
          }
        }
      }
    }
  }
};
// The same for keys key0 .. of the tail (fp16).
template <int D, int NT, int HB>
struct Kv8TailScores {
  TailView tail;
  int key0;
  const uint4* sq;
  int lane;
  __device__ __forceinline__ Kv8TailScores again() const {
    Kv8TailScores q = *this;
    asm volatile("" : "+l"(q.tail.k), "+l"(q.sq));
    return q;
  }
  __device__ __forceinline__ void operator()(float (&s)[HB][NT][4]) const {
    constexpr int NE = D / 64;
#pragma unroll
    for (int b = 0; b < HB; ++b) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[b][n][i] = 0.f;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        uint2 kA[4], kB[4];
        tail_k_frag<D>(tail, key0 + 16 * b, e, lane >> 2, lane & 3, kA, kB);
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 qv = sq[((n * NE + e) * 2 + s2) * 32 + lane];
            const uint32_t f0[4] = {kA[2 * s2].x, kB[2 * s2].x, kA[2 * s2].y, kB[2 * s2].y};
            const uint32_t f1[4] = {kA[2 * s2 + 1].x, kB[2 * s2 + 1].x, kA[2 * s2 + 1].y, kB[2 * s2 + 1].y};
            mma_f16_16816(s[b][n], f0, qv.x, qv.y);
            mma_f16_16816(s[b][n], f1, qv.z, qv.w);
          }
      }
    }
  }
};

// x = x kc + off for one n-tile's scores, masked keys -inf (pos0, pos1: the positions of its rows 2 c and 2 c + 1).
template <int NT, int HB>
__device__ __forceinline__ void kv8_exponents(float (&x)[HB][NT][4], int n, float kc, float2 off, bool open, int pos0, int pos1,
                                              int key, int window) {
#pragma unroll
  for (int b = 0; b < HB; ++b)
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
      const float2 e = ffma2(make_float2(x[b][n][k], x[b][n][k + 1]), make_float2(kc, kc), off);
      x[b][n][k] = e.x;
      x[b][n][k + 1] = e.y;
    }
  if (open) return;
#pragma unroll
  for (int b = 0; b < HB; ++b)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (!sees(pos0, key + 16 * b + 8 * k, window)) x[b][n][2 * k] = -INFINITY;
      if (!sees(pos1, key + 16 * b + 8 * k, window)) x[b][n][2 * k + 1] = -INFINITY;
    }
}

// A warp's running state: O^T accumulators, the maxima of its lanes' rows, the sums of P' / vs, exact and of rounded P'.
template <int D, int NT>
struct Kv8Rows {
  float o[D / 16][NT][4];
  float m[NT][2];
  float2 l[NT], lp[NT];
};

// Softmax of HB x 16 keys from key0 on, P' packed as B operands. qk(x) makes the scores S^T; kc: their factor, lv: log2 of
// the V factor, inv: its reciprocal. The scores become exponents in place; the rare page that moves a maximum makes them
// again (keeping both spills at 16 rows and head_dim 64).
template <int D, int NT, int HB, typename QK>
__device__ __forceinline__ void kv8_softmax(const QK& qk, Kv8Rows<D, NT>& w, const Kv8AttnArgs& a, int row, int key0, bool open,
                                            float kc, float lv, float inv, int lane, uint32_t (&pb)[HB][NT][2]) {
  const int key = key0 + (lane >> 2);
  float x[HB][NT][4];
  qk(x);
  float top = -INFINITY;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = row + 8 * n;
    // +inf against a row without a maximum yet
    kv8_exponents<NT, HB>(x, n, kc, make_float2(lv - w.m[n][0], lv - w.m[n][1]), open, open ? 0 : a.ctx_len + r / a.group,
                          open ? 0 : a.ctx_len + (r + 1) / a.group, key, a.window);
#pragma unroll
    for (int b = 0; b < HB; ++b) top = fmax3(fmax3(top, x[b][n][0], x[b][n][1]), x[b][n][2], x[b][n][3]);
  }
  if (__any_sync(0xffffffffu, top > kLazy + kHeadroom)) {
    qk.again()(x);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = row + 8 * n;
      kv8_exponents<NT, HB>(x, n, kc, make_float2(lv, lv), open, a.ctx_len + r / a.group, a.ctx_len + (r + 1) / a.group, key,
                            a.window);
      float f[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < HB; ++b) mx = fmax3(mx, x[b][n][i], x[b][n][i + 2]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        mx = fmaxf(mx - kHeadroom, w.m[n][i]);
        f[i] = mx == -INFINITY ? 1.f : fast_exp2(w.m[n][i] - mx);   // no key yet: 2^-inf = 0
        w.m[n][i] = mx;
        const float m = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          w.o[d][n][i] *= f[i];
          w.o[d][n][i + 2] *= f[i];
        }
#pragma unroll
        for (int b = 0; b < HB; ++b) {
          x[b][n][i] -= m;
          x[b][n][i + 2] -= m;
        }
      }
      w.l[n] = fmul2(w.l[n], make_float2(f[0], f[1]));
      w.lp[n] = fmul2(w.lp[n], make_float2(f[0], f[1]));
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float2 sum = make_float2(0.f, 0.f), rsum = sum;
#pragma unroll
    for (int b = 0; b < HB; ++b)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float2 p = make_float2(fast_exp2(x[b][n][2 * k]), fast_exp2(x[b][n][2 * k + 1]));
        const float2 r = round11(p);
        sum = fadd2(sum, p);
        rsum = fadd2(rsum, r);
        pb[b][n][k] = movmatrix_trans(pack_half2(r.x, r.y));
      }
    w.l[n] = ffma2(sum, make_float2(inv, inv), w.l[n]);
    w.lp[n] = ffma2(rsum, make_float2(inv, inv), w.lp[n]);
  }
}

// Attention of up to 8 NT query rows of one kv head over a split's pages. Grid (splits, kv heads, row groups).
//
// Each warp streams its own pages (every kWarps-th of the split's) through its own ring of bulk copies, so no warp waits
// for another before the end, and turns codes into fp16 operands in registers: Q, K and P V products are exact to fp32
// accumulation, only P is rounded to fp16. Scores come as S^T (keys x rows), so the sealed pages' K scale is one factor
// per page, and the V scale is folded into the exponent: P' = 2^(s + log2 vs - m'), with m' the running maximum of
// s + log2 vs less kHeadroom, gives sum P' v8 = 2^-m' sum 2^s v directly, and l = sum P' / vs is the softmax sum, of fp32
// P': a page of small vs keeps its share of the sum where its P' is below fp16's normal values (round11). m' is lazy (moved
// only when a score passes it by 2^15; fp16 P then stays within 2^15 and fp32 sums are unaffected), so the common page
// needs no shuffles but one vote. A warp's open pages come last: their factor of 1 moves m' when the others' P' is summed
// already. movmatrix turns the S^T accumulators into the B operand of O^T = V^T P.
// The warps meet in shared memory at the end; one split writes its rows, several write (acc, m', l) partials.
// What bounds it: HBM for one token (100003 tokens at 32/8/64, int8: 21.9 us with the merge, 4.7 TB/s; 131072: 27.0 us),
// instructions from 2 n-tiles on (some 380 a page and warp at 16 rows, 55% of the issue slots with 16 warps per SM).
//
// CLUSTER: the splits of a kv head are a cluster of kKv8Cluster blocks that merge through each other's shared memory, so a
// short context needs no second launch. Over 777 tokens (int8), one launch against two: 32/8/64, 1 token 5.8 us against
// 5.8, 4 tokens 7.2 against 8.4; 16/4/128, 6.6 against 7.1 and 9.4 against 10.7; and 2.3 us less of the host's time each.
constexpr int kKv8Cluster = 8;
template <int D, int NT, bool E4M3, bool CLUSTER>
__device__ __forceinline__ void kv8_attend(const Kv8AttnArgs& a) {
  using L = Kv8Attn<D, NT>;
  using S = Q8Section<D>;
  constexpr int W = L::kWarps, NS = L::kStages, NR = 8 * NT;
  constexpr int HB = 2;   // both 16-key halves of a page together: independent MMA chains, one vote
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int h = blockIdx.y, split = blockIdx.x, row0 = blockIdx.z * NR, rows = a.m * a.group;
  const int kv_end = a.ctx_len + a.m;
  const int pg0 = a.p_begin + (int)((int64_t)a.p_total * split / a.splits);
  const int pg1 = a.p_begin + (int)((int64_t)a.p_total * (split + 1) / a.splits);
  const int sealed_end = min(pg1, a.sealed / kBlockTokens);   // the split's sealed pages are [pg0, sealed_end)
  uint4* sq = reinterpret_cast<uint4*>(smem + L::kOffQ);
  float* sbias = reinterpret_cast<float*>(smem + L::kOffBias);
  uint8_t* ring = smem + (size_t)warp * NS * L::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kOffBar) + warp * NS;

  if (lane == 0) {
    for (int s = 0; s < NS; ++s) mbar_init(&full[s], 1);
    fence_barrier_init();
  }
  __syncwarp();
  pdl_wait();
  const char* head = a.g.pool + h * a.g.head_bytes;
  const int first = pg0 + warp;
  const int npages = first < sealed_end ? (sealed_end - first + W - 1) / W : 0;   // this warp's sealed pages
  // Block-table entries 32 of this warp's pages at a time, one per lane (a load per page would stall the warp).
  int tab0 = 0;
  int64_t entry = 0;
  auto load_entries = [&] { entry = tab0 + lane < npages ? phys_block(a.g, first + (tab0 + lane) * W) : 0; };
  load_entries();
  int issued = 0;
  auto issue = [&](int st) {
    if (issued - tab0 == 32) {
      tab0 += 32;
      load_entries();
    }
    const int64_t blk = __shfl_sync(0xffffffffu, entry, issued - tab0);
    if (lane == 0) {
      mbar_arrive_expect_tx(&full[st], L::kStageBytes);
      bulk_g2s(ring + st * L::kStageBytes, head + blk * a.g.block_bytes, L::kStageBytes, &full[st]);
    }
    ++issued;
  };
  while (issued < min(NS, npages)) issue(issued);
  stage_q<D>(a.q, a.q_stride, rows, a.group, h, row0, NT, sq, threadIdx.x, L::kThreads);
  if (!E4M3)
    stage_bias<D>(a.q, a.q_stride, rows, a.group, h, row0, NR, kCodeBias<E4M3>, sbias, warp, W, lane);
  __syncthreads();

  Kv8Rows<D, NT> w;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    w.m[n][0] = w.m[n][1] = -INFINITY;
    w.l[n] = w.lp[n] = make_float2(0.f, 0.f);
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) w.o[d][n][i] = 0.f;
  }

  const TailView tail = tail_of(a.tail, a.g.kv_heads, h, D);
  bool ok = true;
  int st = 0, waited = 0;
  uint32_t phase = 0;
#pragma unroll 1
  for (; waited < npages;) {
    ok = __all_sync(0xffffffffu, mbar_wait(&full[st], phase));
    if (!ok) break;
    const int page = first + waited * W;
    ++waited;
    const uint8_t* sec = ring + st * L::kStageBytes;
    const float vs = reinterpret_cast<const float*>(sec)[kFactorWord];
    const float kc = reinterpret_cast<const float*>(sec)[0] * kCodeUnit<E4M3> * a.qk_scale, lv = __log2f(vs), inv = __fdividef(1.f, vs);
    const bool open = page_open(page, a.ctx_len, a.m, a.window);
    const Kv8Scores<D, NT, HB, E4M3> qk{sec + S::kOffK, sq, sbias, lane};
    uint32_t pb[HB][NT][2];
    kv8_softmax<D, NT, HB>(qk, w, a, row0 + 2 * c, page * kBlockTokens, open, kc, lv, inv, lane, pb);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int b = 0; b < HB; ++b) {
        const uint4 r = reinterpret_cast<const uint4*>(sec + S::kOffV)[(b * (D / 32) + d) * 32 + lane];
        const uint32_t f0[4] = {decode_pair<E4M3, false>(r.x), decode_pair<E4M3, false>(r.y),
                                decode_pair<E4M3, true>(r.x), decode_pair<E4M3, true>(r.y)};
        const uint32_t f1[4] = {decode_pair<E4M3, false>(r.z), decode_pair<E4M3, false>(r.w),
                                decode_pair<E4M3, true>(r.z), decode_pair<E4M3, true>(r.w)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_f16_16816(w.o[2 * d][n], f0, pb[b][n][0], pb[b][n][1]);
          mma_f16_16816(w.o[2 * d + 1][n], f1, pb[b][n][0], pb[b][n][1]);
        }
      }
    __syncwarp();   // every lane has read the stage
    if (issued < npages) issue(st);
    if (++st == NS) {
      st = 0;
      phase ^= 1;
    }
  }
  if (!ok) {   // give up: raise the error word and drain this warp's own copies (bounded)
    if (lane == 0) raise_error(kErrWaitFull);
    for (; waited < issued; ++waited) {
      (void)mbar_wait(&full[st], phase);
      if (++st == NS) {
        st = 0;
        phase ^= 1;
      }
    }
  }
  // Tail pages (fp16): the first one of this warp's at or past the sealed ones.
#pragma unroll 1
  for (int page = first + npages * W; page < pg1; page += W) {
    const int key0 = page * kBlockTokens;
    const Kv8TailScores<D, NT, HB> qk{tail, key0, sq, lane};
    uint32_t pb[HB][NT][2];
    kv8_softmax<D, NT, HB>(qk, w, a, row0 + 2 * c, key0, false, a.qk_scale, 0.f, 1.f, lane, pb);
#pragma unroll
    for (int b = 0; b < HB; ++b) {
      const int k0 = key0 + 16 * b + 2 * c;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        const int dim = 16 * d + g;
        const uint32_t f[4] = {tail_v_pair(tail, k0, dim, kv_end), tail_v_pair(tail, k0, dim + 8, kv_end),
                               tail_v_pair(tail, k0 + 8, dim, kv_end), tail_v_pair(tail, k0 + 8, dim + 8, kv_end)};
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_f16_16816(w.o[d][n], f, pb[b][n][0], pb[b][n][1]);
      }
    }
  }

  // The warps' rows meet in shared memory: [warp][row][D + 4] acc, then [warp][row] (max, sum).
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int x = 4; x <= 16; x <<= 1) {
      w.l[n] = fadd2(w.l[n], make_float2(__shfl_xor_sync(0xffffffffu, w.l[n].x, x), __shfl_xor_sync(0xffffffffu, w.l[n].y, x)));
      w.lp[n] = fadd2(w.lp[n], make_float2(__shfl_xor_sync(0xffffffffu, w.lp[n].x, x), __shfl_xor_sync(0xffffffffu, w.lp[n].y, x)));
    }
    // acc / lp is the mean over rounded P' (numerator and denominator carry the same roundings); from here on acc is
    // relative to the exact sum, which the log-sum-exp needs
    const float f[2] = {w.lp[n].x > 0.f ? w.l[n].x / w.lp[n].x : 1.f, w.lp[n].y > 0.f ? w.l[n].y / w.lp[n].y : 1.f};
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) w.o[d][n][i] *= f[i & 1];
  }
  __syncthreads();   // the rings are drained
  float* so = reinterpret_cast<float*>(smem);
  float2* sm = reinterpret_cast<float2*>(smem + W * NR * L::kOStride * 4);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 8 * n + 2 * c + i;
      float* dst = so + (warp * NR + r) * L::kOStride + g;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        dst[16 * d] = w.o[d][n][i];
        dst[16 * d + 8] = w.o[d][n][i + 2];
      }
      if (g == 0) sm[warp * NR + r] = make_float2(w.m[n][i], i ? w.l[n].y : w.l[n].x);
    }
  }
  __syncthreads();
  float* fin = reinterpret_cast<float*>(smem + L::kMerge);   // CLUSTER: [row][D + 2] acc, max, sum of this split
  for (int i = threadIdx.x; i < NR * (D / 2); i += L::kThreads) {
    const int r = i / (D / 2), d = 2 * (i % (D / 2)), gr = row0 + r;
    if (gr >= rows) break;
    float2 ml[W];
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      ml[w] = sm[w * NR + r];
      mx = fmaxf(mx, ml[w].x);
    }
    float l = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = ml[w].x == -INFINITY ? 0.f : fast_exp2(ml[w].x - mx);
      const float2 v = *reinterpret_cast<const float2*>(so + (w * NR + r) * L::kOStride + d);
      l = fmaf(f, ml[w].y, l);
      x0 = fmaf(f, v.x, x0);
      x1 = fmaf(f, v.y, x1);
    }
    const int t = gr / a.group, row = t * a.q_heads + h * a.group + (gr - t * a.group);
    if constexpr (CLUSTER) {
      float* dst = fin + r * (D + 2);
      *reinterpret_cast<float2*>(dst + d) = make_float2(x0, x1);
      if (d == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(mx, l);
    } else if (a.splits == 1) {
      const float scale = (l > 0.f ? 1.f / l : 0.f) * sigmoid_gate(a.gate, row);
      *reinterpret_cast<uint32_t*>(a.out + (int64_t)row * D + d) = pack_half2(x0 * scale, x1 * scale);
      if (a.lse && d == 0) a.lse[row] = (mx + log2f(l)) * kLn2;
    } else {
      float* dst = a.part + ((int64_t)row * a.splits + split) * (D + 2);
      *reinterpret_cast<float2*>(dst + d) = make_float2(x0, x1);
      if (d == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(mx, l);
    }
  }
  if constexpr (CLUSTER) {   // each block of the cluster writes its share of the rows' pairs of dims
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int rank = (int)cluster.block_rank(), pairs = min(NR, rows - row0) * (D / 2);
    for (int i = pairs * rank / kKv8Cluster + threadIdx.x; i < pairs * (rank + 1) / kKv8Cluster; i += L::kThreads) {
      const int r = i / (D / 2), d = 2 * (i % (D / 2)), gr = row0 + r;
      float2 ml[kKv8Cluster], v[kKv8Cluster];
      float mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < kKv8Cluster; ++k) {
        const float* src = cluster.map_shared_rank(fin, k) + r * (D + 2);
        ml[k] = *reinterpret_cast<const float2*>(src + D);
        v[k] = *reinterpret_cast<const float2*>(src + d);
        mx = fmaxf(mx, ml[k].x);
      }
      float l = 0.f, x0 = 0.f, x1 = 0.f;
#pragma unroll
      for (int k = 0; k < kKv8Cluster; ++k) {
        const float f = ml[k].x == -INFINITY ? 0.f : fast_exp2(ml[k].x - mx);
        l = fmaf(f, ml[k].y, l);
        x0 = fmaf(f, v[k].x, x0);
        x1 = fmaf(f, v[k].y, x1);
      }
      const int t = gr / a.group, row = t * a.q_heads + h * a.group + (gr - t * a.group);
      const float scale = (l > 0.f ? 1.f / l : 0.f) * sigmoid_gate(a.gate, row);
      *reinterpret_cast<uint32_t*>(a.out + (int64_t)row * D + d) = pack_half2(x0 * scale, x1 * scale);
      if (a.lse && d == 0) a.lse[row] = (mx + log2f(l)) * kLn2;
    }
    cluster.sync();   // no block leaves while another may still read its shared memory
  }
}
template <int D, int NT, bool E4M3>
__global__ __launch_bounds__(Kv8Attn<D, NT>::kThreads, Kv8Attn<D, NT>::kBlocksPerSm) void kv8_attend_kernel(Kv8AttnArgs a) {
  kv8_attend<D, NT, E4M3, false>(a);
}
template <int D, int NT, bool E4M3>
__global__ __cluster_dims__(kKv8Cluster, 1, 1) __launch_bounds__(Kv8Attn<D, NT>::kThreads, Kv8Attn<D, NT>::kBlocksPerSm)
void kv8_attend_cluster_kernel(Kv8AttnArgs a) {
  kv8_attend<D, NT, E4M3, true>(a);
}

// Merge of a row's split partials (acc[D], max, sum): one block of 2 D threads per row, thread = (pair of dims, quarter of
// the splits). The loads of 64 splits go out at once (a lane of each warp holds (max, sum) of two splits): one round trip
// to L2 where maxima, sums and accumulators one after the other took three. More splits go 64 at a time.
constexpr int kKv8MaxSplits = 1024;
template <int D>
__global__ __launch_bounds__(2 * D, 4) void kv8_combine_kernel(const float* part, int splits, const __half* gate, __half* out,
                                                            float* lse) {
  constexpr int P = D / 2, G = 4, U = 64 / G;
  __shared__ float2 acc[G][P];
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.x, tid = threadIdx.x, p = tid % P, gi = tid / P, lane = tid & 31;   // a warp has one gi
  const float* base = part + (int64_t)row * splits * (D + 2);
  float M = -INFINITY, l = 0.f;
  float2 x = make_float2(0.f, 0.f);
  for (int s0 = 0; s0 < splits; s0 += 64) {
    float2 ml[2], v[U];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int s = s0 + lane + 32 * k;
      ml[k] = s < splits ? *reinterpret_cast<const float2*>(base + (int64_t)s * (D + 2) + D) : make_float2(-INFINITY, 0.f);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {   // splits U gi + u of the 64
      const int s = s0 + U * gi + u;
      v[u] = s < splits ? *reinterpret_cast<const float2*>(base + (int64_t)s * (D + 2) + 2 * p) : make_float2(0.f, 0.f);
    }
    float m = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = fmaxf(m, M);
    const float old = M == -INFINITY ? 0.f : fast_exp2(M - m);
    M = m;
    float w[2], sum = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      w[k] = ml[k].x == -INFINITY ? 0.f : fast_exp2(ml[k].x - m);
      sum = fmaf(w[k], ml[k].y, sum);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l = fmaf(l, old, sum);
    x.x *= old;
    x.y *= old;
#pragma unroll
    for (int u = 0; u < U; ++u) {   // all of a warp's splits lie in one half of the 64
      const float f = __shfl_sync(0xffffffffu, gi < G / 2 ? w[0] : w[1], (U * gi + u) & 31);
      x.x = fmaf(f, v[u].x, x.x);
      x.y = fmaf(f, v[u].y, x.y);
    }
  }
  acc[gi][p] = x;
  __syncthreads();
  if (gi == 0) {
#pragma unroll
    for (int k = 1; k < G; ++k) {
      x.x += acc[k][p].x;
      x.y += acc[k][p].y;
    }
    const float scale = (l > 0.f ? 1.f / l : 0.f) * sigmoid_gate(gate, row);
    *reinterpret_cast<uint32_t*>(out + (int64_t)row * D + 2 * p) = pack_half2(x.x * scale, x.y * scale);
    if (lse && p == 0) lse[row] = (M + log2f(l)) * kLn2;
  }
}

// ---------------------------------------------------------------- prefill staging
template <int D>
constexpr int kStagedHeadBytes = F16Section<D>::kOffV8;   // a MODE_F16 section without the int8 V copy: K, then V

struct Kv8ExpandArgs {
  KvGeom g;
  __half* tail;
  char* dst;         // staged sections [page][kv head]
  int32_t* table;    // the staged pages' block table, logical pages page0 .. page0 + grid.x - 1
  float4* scales;    // [page - page0][kv head]: K factor, log2 of the V factor, its reciprocal
  int page0, sealed, len;
};

// One page and kv head of the cache as the K and V tiles of a MODE_F16 section, the codes as fp16 (exactly; the scales go
// beside them): what the prefill kernel's SCALED form reads. Values past the sequence's end are 0. 32000 tokens at 4 heads
// of 128 take 17 us beside 760 for a chunk of 1999 over them; expanding inside the prefill kernel would repeat the work
// for each of the chunk's 63 row tiles.
template <int D, bool E4M3>
__global__ __launch_bounds__(128) void kv8_expand_kernel(Kv8ExpandArgs a) {
  using S = Q8Section<D>;
  using F = F16Section<D>;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, page = a.page0 + blockIdx.x, h = blockIdx.y, t0 = page * kBlockTokens;
  if (h == 0 && tid == 0) a.table[page] = blockIdx.x;
  const int64_t section = (int64_t)blockIdx.x * a.g.kv_heads + h;
  char* dst = a.dst + section * kStagedHeadBytes<D>;
  uint4* K = reinterpret_cast<uint4*>(dst);
  uint4* V = reinterpret_cast<uint4*>(dst + F::kOffV);
  if (t0 < a.sealed) {
    const char* sec = a.g.pool + phys_block(a.g, page) * a.g.block_bytes + h * a.g.head_bytes;
    if (tid == 0) {
      const float ks = reinterpret_cast<const float*>(sec)[0];
      const float vs = reinterpret_cast<const float*>(sec)[kFactorWord];
      a.scales[section] = make_float4(ks, log2f(vs), 1.f / vs, 0.f);
    }
    // Tile rows of 16 bytes: 8 dims of one key (K), 8 keys of one dim (V).
    for (int i = tid; i < 2 * D; i += 128) {
      const int l = i & 31, b = i >> 5;
      const int key = (b / (D / 64)) * 8 + (l >> 2), d8 = (b % (D / 64)) * 8 + (l & 3) * 2;
      const uint4 w = reinterpret_cast<const uint4*>(sec + S::kOffK)[i];
      uint4* dst = K + ((key >> 3) * (D / 8) + d8) * 8 + (key & 7);
      dst[0] = make_uint4(decode_pair<E4M3, false>(w.x), decode_pair<E4M3, true>(w.x), decode_pair<E4M3, false>(w.y),
                          decode_pair<E4M3, true>(w.y));
      dst[8] = make_uint4(decode_pair<E4M3, false>(w.z), decode_pair<E4M3, true>(w.z), decode_pair<E4M3, false>(w.w),
                          decode_pair<E4M3, true>(w.w));
    }
    const uint32_t* V4 = reinterpret_cast<const uint32_t*>(sec + S::kOffV);
    for (int i = tid; i < 2 * D; i += 128) {   // 16 keys of one dim: four words
      const int wi = i & 3, g = (i >> 2) & 7, dtp = (i >> 5) % (D / 32), mt = (i >> 5) / (D / 32);
      const int d = 32 * dtp + 16 * (wi >> 1) + 8 * (wi & 1) + g;
      uint32_t w[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) w[c] = V4[S::v_index(16 * mt + 2 * c, d) / 4];
      uint4* dst = V + ((d >> 3) * 4 + 2 * mt) * 8 + (d & 7);
      dst[0] = make_uint4(decode_pair<E4M3, false>(w[0]), decode_pair<E4M3, false>(w[1]), decode_pair<E4M3, false>(w[2]),
                          decode_pair<E4M3, false>(w[3]));
      dst[8] = make_uint4(decode_pair<E4M3, true>(w[0]), decode_pair<E4M3, true>(w[1]), decode_pair<E4M3, true>(w[2]),
                          decode_pair<E4M3, true>(w[3]));
    }
    return;
  }
  const TailView tail = tail_of(a.tail, a.g.kv_heads, h, D);
  if (tid == 0) a.scales[section] = make_float4(1.f, 0.f, 1.f, 0.f);
  for (int i = tid; i < 4 * D; i += 128) {
    const int e = i & 7, tile = i >> 3;
    const int key = (tile / (D / 8)) * 8 + e, d = (tile % (D / 8)) * 8;
    K[i] = t0 + key < a.len ? *reinterpret_cast<const uint4*>(tail.k + (int64_t)((t0 + key) % kTailTokens) * D + d)
                            : make_uint4(0, 0, 0, 0);
    const int vd = (tile >> 2) * 8 + e, key0 = (tile & 3) * 8;
    uint32_t v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      v[k] = t0 + key0 + 2 * k < a.len ? tail_v_pair(tail, t0 + key0 + 2 * k, vd, a.len) : 0u;
    V[i] = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

// ---------------------------------------------------------------- attention weights per key
struct Kv8WeightArgs {
  KvGeom g;
  __half* tail;
  const __half* q;
  const float* lse;     // [m][q_heads]
  const float* prev;    // [kv_heads][stride], or null
  float* out;           // [kv_heads][stride]
  int64_t q_stride, prev_stride, out_stride;
  int m, group, q_heads, ctx_len, window, sealed, splits, pages;
  float decay, qk_scale;
};

template <int D>
struct Kv8Weights {
  static constexpr int kWarps = 8, kThreads = 32 * kWarps, kStages = D == 64 ? 4 : 2;
  static constexpr int kStageBytes = Q8Section<D>::kOffV;   // the header and K
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kMaxRows = 256;
  static __host__ __device__ constexpr int lse_off(int ntiles) { return kRing + ntiles * 8 * D * 2; }
  static __host__ __device__ constexpr int bias_off(int ntiles) { return lse_off(ntiles) + ntiles * 8 * 4; }
  static __host__ __device__ constexpr int bar_off(int ntiles) { return bias_off(ntiles) + ntiles * 8 * 4; }
  static __host__ __device__ constexpr int part_off(int ntiles) { return bar_off(ntiles) + kWarps * kStages * 8; }
  static __host__ __device__ constexpr int smem(int ntiles) { return part_off(ntiles) + kThreads * 4; }
};

// out[h][key] = decay prev[h][key] + sum over the m tokens and the head's query rows of 2^(s - lse): only K is read. A
// warp takes a page (as kv8_attend_kernel does), makes its K operands once and passes over the query rows 8 at a time, two
// independent chains of MMAs (16 keys each) per 8 rows; a lane owns the weights of 4 keys for 2 rows in 8, so the sums
// meet in two shuffles per page and no atomics are needed. prev is loaded a page ahead (loaded when wanted, its latency
// was two thirds of the time of a single token's pass). Grid (splits, kv heads). Bound by HBM and the latency of a page's
// chain of MMAs for one token (131072 tokens at 32/8/64: 19.2 us with a sum so far, 3.9 TB/s), by the MMAs for many rows.
// SHARE: in a last round with half of a block's warps or less to do, 2 to 8 warps share a page's rows, and their sums meet
// in shared memory. It costs the loop some instructions: int8, 32/8/64, 32 tokens over 20000 17.0 us against 19.1 without
// (2 rounds of pages), 4 tokens over 131000 22.8 against 20.5 (14 rounds), so kv8_weights_share picks it for few rounds.
template <int D, bool E4M3, bool SHARE>
__global__ __launch_bounds__(Kv8Weights<D>::kThreads, 2) void kv8_weights_kernel(Kv8WeightArgs a) {
  using L = Kv8Weights<D>;
  using S = Q8Section<D>;
  constexpr int NE = D / 64, W = L::kWarps, NS = L::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int h = blockIdx.y, rows = a.m * a.group, ntiles = (rows + 7) / 8, kv_end = a.ctx_len + a.m;
  const int pg0 = (int)((int64_t)a.pages * blockIdx.x / a.splits), pg1 = (int)((int64_t)a.pages * (blockIdx.x + 1) / a.splits);
  const int sealed_pages = a.sealed / kBlockTokens;
  uint4* sq = reinterpret_cast<uint4*>(smem + L::kRing);
  float* slse = reinterpret_cast<float*>(smem + L::lse_off(ntiles));
  float* sbias = reinterpret_cast<float*>(smem + L::bias_off(ntiles));
  uint8_t* ring = smem + (size_t)warp * NS * L::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::bar_off(ntiles)) + warp * NS;

  if (lane == 0) {
    for (int s = 0; s < NS; ++s) mbar_init(&full[s], 1);
    fence_barrier_init();
  }
  __syncwarp();
  pdl_wait();
  const char* head = a.g.pool + h * a.g.head_bytes;
  auto issue = [&](int page, int st) {
    mbar_arrive_expect_tx(&full[st], L::kStageBytes);
    bulk_g2s(ring + st * L::kStageBytes, head + phys_block(a.g, page) * a.g.block_bytes, L::kStageBytes, &full[st]);
  };
  // This warp's pages in order: one of each 8; of a last round with half of the warps or less to do, a share of the rows.
  const int whole = (pg1 - pg0) / W, rest = (pg1 - pg0) % W;
  int share = !SHARE || rest == 0 || rest > W / 2 ? 1 : rest == 1 ? 8 : rest == 2 ? 4 : 2;   // warps to a page of the last round
  if (SHARE)
    while (share > ntiles) share /= 2;
  const int last = min(pg1, pg0 + whole * W + warp / share), sub = SHARE ? warp % share : 0;
  auto page_of = [&](int k) {   // pg1 or more past the last one
    return !SHARE || k < whole ? pg0 + k * W + warp : k == whole ? last : pg1;
  };
  const int end = min(pg1, sealed_pages);
  int issued = 0, waited = 0;
  while (issued < NS && page_of(issued) < end) {
    if (lane == 0) issue(page_of(issued), issued);
    ++issued;
  }
  stage_q<D>(a.q, a.q_stride, rows, a.group, h, 0, ntiles, sq, threadIdx.x, L::kThreads);
  if (!E4M3) stage_bias<D>(a.q, a.q_stride, rows, a.group, h, 0, 8 * ntiles, kCodeBias<E4M3>, sbias, warp, W, lane);
  for (int r = threadIdx.x; r < 8 * ntiles; r += L::kThreads) {
    const int t = r / a.group, j = r - t * a.group;
    // a padding row, and a row that saw no key (lse -inf), weighs nothing
    float x = r < rows ? a.lse[t * a.q_heads + h * a.group + j] * kLog2e : INFINITY;
    slse[r] = x == -INFINITY ? INFINITY : x;
  }
  __syncthreads();

  const TailView tail = tail_of(a.tail, a.g.kv_heads, h, D);
  float* spart = reinterpret_cast<float*>(smem + L::part_off(ntiles));
  // The page's 32 keys against all rows, or a share of them; lane i adds key i's sum to old and stores it.
  auto rows32 = [&](const uint32_t (&f)[2][4 * NE][4], int page, bool shared, bool open, float kc, float old, bool biased) {
    float w[4] = {0.f, 0.f, 0.f, 0.f};   // keys 8 i + g
#pragma unroll 2
    for (int n = SHARE && shared ? sub : 0; n < ntiles; n += SHARE && shared ? share : 1) {
      float2 bias = make_float2(0.f, 0.f);
      if (!E4M3 && biased) bias = *reinterpret_cast<const float2*>(sbias + 8 * n + 2 * c);
      float s[2][4] = {{bias.x, bias.y, bias.x, bias.y}, {bias.x, bias.y, bias.x, bias.y}};
#pragma unroll
      for (int e = 0; e < 2 * NE; ++e) {
        const uint4 qv = sq[(n * 2 * NE + e) * 32 + lane];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) mma_f16_16816(s[mt], f[mt][2 * e], qv.x, qv.y);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) mma_f16_16816(s[mt], f[mt][2 * e + 1], qv.z, qv.w);
      }
      const float2 z = *reinterpret_cast<const float2*>(slse + 8 * n + 2 * c);
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = fast_exp2(fmaf(s[mt][i], kc, (i & 1) ? -z.y : -z.x));
        if (!open) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int pos = a.ctx_len + (8 * n + 2 * c + (i & 1)) / a.group;
            if (!sees(pos, page * kBlockTokens + 16 * mt + g + 8 * (i >> 1), a.window)) p[i] = 0.f;
          }
        }
        w[2 * mt] += p[0] + p[1];
        w[2 * mt + 1] += p[2] + p[3];
      }
    }
    float mine = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] += __shfl_xor_sync(0xffffffffu, w[i], 1);
      w[i] += __shfl_xor_sync(0xffffffffu, w[i], 2);
      const float v = __shfl_sync(0xffffffffu, w[i], 4 * (lane & 7));   // key 8 i + lane % 8
      if ((lane >> 3) == i) mine = v;
    }
    const int key = page * kBlockTokens + lane;
    if (SHARE && shared) spart[warp * 32 + lane] = mine;
    else if (key < kv_end) a.out[h * a.out_stride + key] = fmaf(a.decay, old, mine);
  };
  auto load_prev = [&](int page) -> float {
    const int key = page * kBlockTokens + lane;
    return a.prev && page < pg1 && key < kv_end ? a.prev[h * a.prev_stride + key] : 0.f;
  };

  float old_next = load_prev(page_of(0));
  bool ok = true;
  int st = 0, k = 0;
  uint32_t phase = 0;
  for (; page_of(k) < end; ++k) {
    const int page = page_of(k);
    ok = __all_sync(0xffffffffu, mbar_wait(&full[st], phase));
    if (!ok) break;
    ++waited;
    const uint8_t* sec = ring + st * L::kStageBytes;
    const float kc = reinterpret_cast<const float*>(sec)[0] * kCodeUnit<E4M3> * a.qk_scale;
    const bool open = page_open(page, a.ctx_len, a.m, a.window);
    const float old = old_next;
    old_next = load_prev(page_of(k + 1));
    uint32_t f[2][4 * NE][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const uint4* kc4 = reinterpret_cast<const uint4*>(sec + S::kOffK) + (mt * 2 * NE) * 32 + lane;
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const uint4 ra = kc4[e * 32], rb = kc4[(NE + e) * 32];
        const uint32_t wa[4] = {ra.x, ra.y, ra.z, ra.w}, wb[4] = {rb.x, rb.y, rb.z, rb.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          f[mt][4 * e + u][0] = decode_raw<E4M3, false>(wa[u]);
          f[mt][4 * e + u][1] = decode_raw<E4M3, false>(wb[u]);
          f[mt][4 * e + u][2] = decode_raw<E4M3, true>(wa[u]);
          f[mt][4 * e + u][3] = decode_raw<E4M3, true>(wb[u]);
        }
      }
    }
    rows32(f, page, SHARE && share > 1 && k == whole, open, kc, old, true);
    __syncwarp();
    if (page_of(issued) < end) {
      if (lane == 0) issue(page_of(issued), st);
      ++issued;
    }
    if (++st == NS) {
      st = 0;
      phase ^= 1;
    }
  }
  if (!ok) {
    if (lane == 0) raise_error(kErrWaitFull);
    for (; waited < issued; ++waited) {
      (void)mbar_wait(&full[st], phase);
      if (++st == NS) {
        st = 0;
        phase ^= 1;
      }
    }
  }
  for (; ok && page_of(k) < pg1; ++k) {
    const int page = page_of(k);
    uint32_t f[2][4 * NE][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        uint2 kA[4], kB[4];
        tail_k_frag<D>(tail, page * kBlockTokens + 16 * mt, e, g, c, kA, kB);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          f[mt][4 * e + u][0] = kA[u].x;
          f[mt][4 * e + u][1] = kB[u].x;
          f[mt][4 * e + u][2] = kA[u].y;
          f[mt][4 * e + u][3] = kB[u].y;
        }
      }
    rows32(f, page, SHARE && share > 1 && k == whole, false, a.qk_scale, load_prev(page), false);
  }
  if (SHARE && share > 1) {   // the shares of the last round's pages meet, in the warps' order
    __syncthreads();
    const int key = last * kBlockTokens + lane;
    if (sub == 0 && last < pg1 && key < kv_end) {
      float sum = 0.f;
      for (int i = 0; i < share; ++i) sum += spart[(warp + i) * 32 + lane];
      a.out[h * a.out_stride + key] = fmaf(a.decay, load_prev(last), sum);
    }
  }
}

}  // namespace lfm3a
