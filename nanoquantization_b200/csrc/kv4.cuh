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

// A head's 128 values, held by 16 neighbouring lanes (half of a warp, all of whose lanes call this): lane l has dimensions 4 l .. + 3
// in a and 64 + 4 l .. + 3 in b.  Gives lane l word l of the row and every lane the parameters of both groups.
template <bool BF16> __device__ __forceinline__ void quantise(const float (&a)[4], const float (&b)[4], uint32_t& word, uint2& params) {
  const int l = threadIdx.x & 15;
  float lo[2] = {min_nan(min_nan(a[0], a[1]), min_nan(a[2], a[3])), min_nan(min_nan(b[0], b[1]), min_nan(b[2], b[3]))};
  float hi[2] = {max_nan(max_nan(a[0], a[1]), max_nan(a[2], a[3])), max_nan(max_nan(b[0], b[1]), max_nan(b[2], b[3]))};
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      lo[g] = min_nan(lo[g], __shfl_xor_sync(0xFFFFFFFFu, lo[g], o));
      hi[g] = max_nan(hi[g], __shfl_xor_sync(0xFFFFFFFFu, hi[g], o));
    }
  }
  params = make_uint2(group_params<BF16>(lo[0], hi[0]), group_params<BF16>(lo[1], hi[1]));
  uint32_t part[2];      // this lane's four nibbles of each group's word: of its places 0, 4, 1, 5 in an even lane, 2, 6, 3, 7 in an odd one
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const uint32_t p = g ? params.y : params.x;
    // A true division: values and parameters of few bits often lie exactly between two levels, where a reciprocal's rounding would
    // decide (the values of 4096 bfloat16 tokens: 0.0025 off the true ones in the 2-norm with it, 0.0017 so).
    const float s = scale_of<BF16>(p), m = offset_of<BF16>(p);
    uint32_t n[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) n[e] = s > 0.f ? (uint32_t)fminf(fmaxf(rintf(__fdiv_rn((g ? b[e] : a[e]) - m, s)), 0.f), 15.f) : 0u;
    part[g] = (n[0] | (n[1] << 16) | (n[2] << 4) | (n[3] << 20)) << (8 * (l & 1));
  }
  // even lanes keep group 0 and odd ones group 1
  const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, (l & 1) ? part[0] : part[1], 1);
  word = ((l & 1) ? part[1] : part[0]) | got;
}

// A level as a 16-bit number.  The highest one may lie beyond the type's largest number by the scale's rounding: it is that number.
template <bool BF16> __device__ __forceinline__ uint16_t level(float n, float scale, float offset) {
  constexpr float kTop = BF16 ? 3.3895313892515355e38f : 65504.f;
  return float_to_raw16<BF16>(min_nan(max_nan(fmaf(n, scale, offset), -kTop), kTop));
}

__device__ __forceinline__ float nibble(uint32_t word, int i) { return (float)((word >> (4 * i)) & 15u); }

}  // namespace kv4
}  // namespace nqb200
