// The 4-bit key/value cache: where a row lies, and how 128 values become one.  The layout is stated at nqb200_kv4.
#pragma once
#include "common.cuh"

namespace nqb200 {
namespace kv4 {

constexpr int kDim = 128, kGroup = 64, kData = 64, kParams = 8, kToken = kData + kParams;   // bytes of a row: nibbles; scales and offsets

struct Cache {
  uint8_t *k, *v;
  int64_t pages;
  int kv_heads, block;
};

static inline int check_cache(const nqb200_kv4* c) {
  if (!c) return NQB200_ERR_NULL_POINTER;
  if (c->pages <= 0 || c->pages > INT32_MAX || c->kv_heads <= 0 || c->kv_heads > 4096 || c->block_size <= 0 || c->block_size % 16 != 0 || c->block_size > (1 << 20))
    return NQB200_ERR_BAD_SHAPE;
  if (!c->k || !c->v) return NQB200_ERR_NULL_POINTER;
  return aligned16(c->k) && aligned16(c->v) ? NQB200_OK : NQB200_ERR_MISALIGNED;
}
static inline Cache cache_of(const nqb200_kv4* c) { return Cache{(uint8_t*)c->k, (uint8_t*)c->v, c->pages, (int)c->kv_heads, (int)c->block_size}; }

// Byte offset of a page's share of a head.
__device__ __forceinline__ int64_t page_at(const Cache& c, int64_t page, int head) { return (page * c.kv_heads + head) * ((int64_t)c.block * kToken); }

__device__ __forceinline__ void report(int* status, int code) {
  if (status) atomicExch(status, code);
}

// Minimum and maximum that a NaN does not get lost in.
__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// Scale and offset of a group from its smallest and largest value: two 16-bit numbers, scale first.
template <bool BF16> __device__ __forceinline__ uint32_t group_params(float lo, float hi) {
  const uint16_t m = float_to_raw16<BF16>(lo);
  const float d = hi - raw16_to_float<BF16>(m);
  const uint16_t s = float_to_raw16<BF16>(fabsf(d) < INFINITY ? d / 15.f : __int_as_float(0x7FC00000));
  return (uint32_t)s | ((uint32_t)m << 16);
}
template <bool BF16> __device__ __forceinline__ float scale_of(uint32_t params) { return raw16_to_float<BF16>((uint16_t)(params & 0xFFFF)); }
template <bool BF16> __device__ __forceinline__ float offset_of(uint32_t params) { return raw16_to_float<BF16>((uint16_t)(params >> 16)); }

// A head's 128 values are held by 8 neighbouring lanes, lane m of them dimensions 8 m .. + 7 in x and 64 + 8 m .. + 7 in y: what a rotation pairs
// lies in one lane, the two halves are the two groups of a row, and words 2 m and 2 m + 1 of the row are the lane's own.  All
// lanes of the warp call these.

template <bool BF16> __device__ __forceinline__ void unpack8(uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = raw16_to_float<BF16>((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
}

// (rows of 16 bytes, or where the heads start on 8 bytes only, of two times 8)
template <bool WIDE> __device__ __forceinline__ uint4 fetch8(const uint16_t* src, int piece) {
  if (WIDE) return reinterpret_cast<const uint4*>(src)[piece];
  const uint2 a = reinterpret_cast<const uint2*>(src)[2 * piece], b = reinterpret_cast<const uint2*>(src)[2 * piece + 1];
  return make_uint4(a.x, a.y, b.x, b.y);
}

// A head of projections: RMS norm with `weight` and rotation by `angles` (cos of the 64 pairs, then sin), in float; `weight` null: as it is.
template <bool BF16, bool WIDE = true>
__device__ __forceinline__ void head_values(const uint16_t* src, const uint16_t* weight, const float* angles, float eps, float (&x)[8], float (&y)[8]) {
  const int m = threadIdx.x & 7;
  const uint4 lo = fetch8<WIDE>(src, m), hi = fetch8<WIDE>(src, m + 8);
  uint4 wl = make_uint4(0u, 0u, 0u, 0u), wh = wl;
  float4 c[2], s[2];
  if (weight) {
    wl = fetch8<WIDE>(weight, m);
    wh = fetch8<WIDE>(weight, m + 8);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      c[k] = reinterpret_cast<const float4*>(angles)[2 * m + k];
      s[k] = reinterpret_cast<const float4*>(angles)[16 + 2 * m + k];
    }
  }
  unpack8<BF16>(lo, x);
  unpack8<BF16>(hi, y);
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += x[e] * x[e] + y[e] * y[e];
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
  if (!weight) return;
  const float inv = rsqrtf(ss / (float)kDim + eps);
  float a[8], b[8];
  unpack8<BF16>(wl, a);
  unpack8<BF16>(wh, b);
  const float cv[8] = {c[0].x, c[0].y, c[0].z, c[0].w, c[1].x, c[1].y, c[1].z, c[1].w}, sv[8] = {s[0].x, s[0].y, s[0].z, s[0].w, s[1].x, s[1].y, s[1].z, s[1].w};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float u = x[e] * inv * a[e], v = y[e] * inv * b[e];
    x[e] = u * cv[e] - v * sv[e];
    y[e] = u * sv[e] + v * cv[e];
  }
}

// Words 2 m and 2 m + 1 of the row, and the parameters of both groups in every lane.
template <bool BF16> __device__ __forceinline__ void quantise(const float (&x)[8], const float (&y)[8], uint2& words, uint2& params) {
  float lo[2] = {x[0], y[0]}, hi[2] = {x[0], y[0]};
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    lo[0] = min_nan(lo[0], x[e]); hi[0] = max_nan(hi[0], x[e]);
    lo[1] = min_nan(lo[1], y[e]); hi[1] = max_nan(hi[1], y[e]);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      lo[g] = min_nan(lo[g], __shfl_xor_sync(0xFFFFFFFFu, lo[g], o));
      hi[g] = max_nan(hi[g], __shfl_xor_sync(0xFFFFFFFFu, hi[g], o));
    }
  }
  params = make_uint2(group_params<BF16>(lo[0], hi[0]), group_params<BF16>(lo[1], hi[1]));
  uint32_t word[2] = {0u, 0u};
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    // The product with the reciprocal decides unless it lies near the middle between two levels, where the true quotient does: values and
    // parameters of few bits often lie exactly there (the values of 4096 bfloat16 tokens: 0.0025 off the true ones in the 2-norm without it,
    // 0.0017 with it).
    const uint32_t p = g ? params.y : params.x;
    const float s = scale_of<BF16>(p), m = offset_of<BF16>(p), inv = s > 0.f ? 1.f / s : 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = (g ? y[e] : x[e]) - m, t = d * inv;
      float n = rintf(t);
      if (fabsf(t - n) > 0.4999f) n = rintf(__fdiv_rn(d, s));
      word[g] |= (uint32_t)fminf(fmaxf(n, 0.f), 15.f) << (4 * (e >> 1) + 16 * (e & 1));
    }
  }
  words = make_uint2(word[0], word[1]);
}

// A level as a 16-bit number.  The highest one may lie beyond the type's largest number by the scale's rounding: it is that number.
template <bool BF16> __device__ __forceinline__ uint16_t level(float n, float scale, float offset) {
  constexpr float kTop = BF16 ? 3.3895313892515355e38f : 65504.f;
  return float_to_raw16<BF16>(min_nan(max_nan(fmaf(n, scale, offset), -kTop), kTop));
}

__device__ __forceinline__ float nibble(uint32_t word, int i) { return (float)((word >> (4 * i)) & 15u); }

}  // namespace kv4
}  // namespace nqb200
