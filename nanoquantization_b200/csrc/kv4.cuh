// The 4-bit key/value cache: where a row lies, and how 128 values become one.  The layout is stated at nqb200_kv4.
#pragma once
#include "common.cuh"
#include "pairs.cuh"

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

// a / b from an approximate reciprocal and one Newton step on the quotient, whose remainder is exact: right where the quotient has few bits.
__device__ __forceinline__ float divided(float a, float b, float reciprocal) {
  const float t = a * reciprocal;
  return fmaf(fmaf(-t, b, a), reciprocal, t);
}
// Scale and offset of a group from its smallest and largest value: two 16-bit numbers, scale first.  (An offset that its rounding put above the
// largest value leaves a scale of 0: all levels are the offset.)
template <bool BF16> __device__ __forceinline__ uint32_t group_params(float lo, float hi) {
  const uint16_t m = float_to_raw16<BF16>(lo);
  const float d = hi - raw16_to_float<BF16>(m);
  const uint16_t s = float_to_raw16<BF16>(fabsf(d) < INFINITY ? fmaxf(divided(d, 15.f, 1.f / 15.f), 0.f) : __int_as_float(0x7FC00000));
  return (uint32_t)s | ((uint32_t)m << 16);
}
template <bool BF16> __device__ __forceinline__ float scale_of(uint32_t params) { return raw16_to_float<BF16>((uint16_t)(params & 0xFFFF)); }
template <bool BF16> __device__ __forceinline__ float offset_of(uint32_t params) { return raw16_to_float<BF16>((uint16_t)(params >> 16)); }

// A head's 128 values are held by 8 neighbouring lanes, lane m of them dimensions 8 m .. + 7 and 64 + 8 m .. + 7, as pairs: what a rotation
// turns together lies in one lane, the two halves are the two groups of a row, and words 2 m and 2 m + 1 of the row are the
// lane's own.  All lanes of the warp call these.
struct Half { uint64_t v[4]; };                 // 8 values

template <bool BF16> __device__ __forceinline__ Half unpack8(uint4 raw) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  Half h;
#pragma unroll
  for (int e = 0; e < 4; ++e) h.v[e] = pair2(raw16_to_float<BF16>((uint16_t)(w[e] & 0xFFFF)), raw16_to_float<BF16>((uint16_t)(w[e] >> 16)));
  return h;
}
__device__ __forceinline__ void values(const Half& h, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) unpair2(h.v[e], x[2 * e], x[2 * e + 1]);
}
template <bool BF16> __device__ __forceinline__ uint4 pack8(const Half& h) {
  float x[8];
  values(h, x);
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (BF16) { const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]); w[e] = *reinterpret_cast<const uint32_t*>(&v); }
    else { const __half2 v = __floats2half2_rn(x[2 * e], x[2 * e + 1]); w[e] = *reinterpret_cast<const uint32_t*>(&v); }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// (rows of 16 bytes, or where the heads start on 8 bytes only, of two times 8)
template <bool WIDE> __device__ __forceinline__ uint4 fetch8(const uint16_t* src, int piece) {
  if (WIDE) return reinterpret_cast<const uint4*>(src)[piece];
  const uint2 a = reinterpret_cast<const uint2*>(src)[2 * piece], b = reinterpret_cast<const uint2*>(src)[2 * piece + 1];
  return make_uint4(a.x, a.y, b.x, b.y);
}

struct Angles { Half c, s; };                   // of the lane's eight pairs
__device__ __forceinline__ Angles angles_of(const float* cos_sin) {      // cos of the 64 pairs, then sin
  const int m = threadIdx.x & 7;
  Angles a;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const ulonglong2 c = reinterpret_cast<const ulonglong2*>(cos_sin)[2 * m + k], s = reinterpret_cast<const ulonglong2*>(cos_sin)[16 + 2 * m + k];
    a.c.v[2 * k] = c.x; a.c.v[2 * k + 1] = c.y;
    a.s.v[2 * k] = s.x; a.s.v[2 * k + 1] = s.y;
  }
  return a;
}
// RMS norm with the weights wx, wy and rotation, in float.  (A lane whose head is a value's takes part in the sum and keeps what it has.)
template <bool BF16>
__device__ __forceinline__ void norm_turn(Half& x, Half& y, uint4 wx, uint4 wy, const Angles& a, float eps, bool turns) {
  uint64_t ss = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) ss = fma2(y.v[e], y.v[e], fma2(x.v[e], x.v[e], ss));
  float s0, s1;
  unpair2(ss, s0, s1);
  s0 += s1;
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) s0 += __shfl_xor_sync(0xFFFFFFFFu, s0, o);
  if (!turns) return;
  const float inv = rsqrtf(s0 / (float)kDim + eps);
  const uint64_t inv2 = pair2(inv, inv), minus = pair2(-1.f, -1.f);
  const Half wa = unpack8<BF16>(wx), wb = unpack8<BF16>(wy);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint64_t u = mul2(mul2(x.v[e], inv2), wa.v[e]), v = mul2(mul2(y.v[e], inv2), wb.v[e]);
    x.v[e] = fma2(u, a.c.v[e], mul2(mul2(v, minus), a.s.v[e]));
    y.v[e] = fma2(u, a.s.v[e], mul2(v, a.c.v[e]));
  }
}

// Words 2 m and 2 m + 1 of the row, and the parameters of both groups in every lane.
template <bool BF16> __device__ __forceinline__ void quantise(const Half& hx, const Half& hy, uint2& words, uint2& params) {
  float v[2][8], lo[2], hi[2];
  values(hx, v[0]);
  values(hy, v[1]);
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    lo[g] = hi[g] = v[g][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) { lo[g] = min_nan(lo[g], v[g][e]); hi[g] = max_nan(hi[g], v[g][e]); }
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
  constexpr float kRound = 12582912.f;          // 1.5 * 2^23: adding it rounds to a whole number, to the even one in the middle
  uint32_t word[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const uint32_t p = g ? params.y : params.x;
    const float s = scale_of<BF16>(p), m = offset_of<BF16>(p);
    // The quotient has to be right where it lies in the middle between two levels, as it often does for values of few bits (the values of 4096
    // bfloat16 tokens: 0.0025 off the true ones in the 2-norm with the reciprocal's product alone, 0.0017 so).  A scale whose reciprocal
    // would overflow takes the true division.
    const float inv = s > 1e-37f ? 1.f / s : 0.f;
    const uint64_t m2 = pair2(-m, -m), inv2 = pair2(inv, inv), s2 = pair2(-s, -s), round2 = pair2(kRound, kRound), back2 = pair2(-kRound, -kRound), shift2 = pair2(16.f, 16.f);
    uint64_t n[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint64_t d = add2((g ? hy : hx).v[e], m2), t = mul2(d, inv2);
      float a, b;
      unpair2(fma2(fma2(t, s2, d), inv2, t), a, b);
      if (s > 0.f && s <= 1e-37f) {
        unpair2(d, a, b);
        a = __fdiv_rn(a, s);
        b = __fdiv_rn(b, s);
      }
      n[e] = add2(add2(pair2(fminf(fmaxf(a, 0.f), 15.f), fminf(fmaxf(b, 0.f), 15.f)), round2), back2);      // (a NaN becomes 0; its scale is one)
    }
    // four nibbles in a float, whose whole numbers are exact: the even dimensions' and the odd ones'
    float even, odd;
    unpair2(add2(fma2(fma2(fma2(n[3], shift2, n[2]), shift2, n[1]), shift2, n[0]), pair2(8388608.f, 8388608.f)), even, odd);
    word[g] = __byte_perm(__float_as_uint(even), __float_as_uint(odd), 0x5410);
  }
  words = make_uint2(word[0], word[1]);
}

// A level within the type's numbers: the highest one may lie beyond the largest by the scale's rounding, and is that number then.
template <bool BF16> __device__ __forceinline__ float level(float n, float scale, float offset) {
  constexpr float kTop = BF16 ? 3.3895313892515355e38f : 65504.f;
  return min_nan(max_nan(fmaf(n, scale, offset), -kTop), kTop);
}

__device__ __forceinline__ float nibble(uint32_t word, int i) { return (float)((word >> (4 * i)) & 15u); }

}  // namespace kv4
}  // namespace nqb200
