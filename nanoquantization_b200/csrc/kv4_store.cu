// Store and read-back of the 4-bit key/value cache.
//
// Both are bound by memory: a token's projections in (256 bytes a head), its queries out and 144 bytes per key/value head stored.
// Eight lanes per (token, head), every access 16 bytes wide (8 where a row of nibbles is written).
//
// 4096 tokens of 32 + 8 + 8 heads, bfloat16 (91 MB, 13.9 us at the copy rate): 22.3 us, 4.1 TB/s (five blocks to an SM 23.4, four 25.0); 100
// tokens of 16 + 8 + 8 2.7.  Issue slots are 64 %
// busy (308 warp instructions for four heads), the ALU 48 %.  16 lanes a head with half the width took 38.5, this with plain arithmetic
// and conversions 32.8, two heads per eight lanes 38.3 (88 registers a thread instead of 48).  Read-back of 4096 rows: 8.9 us (43 MB).
#include "kv4.cuh"

namespace nqb200 {
namespace {

using namespace kv4;

struct StoreArgs {
  const uint16_t* qkv; int64_t stride;
  const uint16_t *qw, *kw;
  const float* cos_sin; int64_t max_positions;
  const int64_t *positions, *rows;
  Cache cache;
  uint16_t* q_out;
  int T, heads;
  float eps;
  int* status;
};

template <bool BF16, bool WIDE>
__global__ void __launch_bounds__(256, 6) kv4_store_kernel(const __grid_constant__ StoreArgs a) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int m = threadIdx.x & 7, Hq = a.heads, Hkv = a.cache.kv_heads, per = Hq + 2 * Hkv;
  const int at = blockIdx.x * 32 + (threadIdx.x >> 3);
  const bool in = at < a.T * per;                      // no early return: other heads of the warp may be inside
  const int t = in ? at / per : 0, hd = in ? at - t * per : 0;
  const bool is_v = hd >= Hq + Hkv, is_q = hd < Hq;
  int64_t pos = a.positions[t];
  const uint16_t *src = a.qkv + (int64_t)t * a.stride + (int64_t)hd * kDim, *weight = is_q ? a.qw : a.kw;
  const uint4 rx = fetch8<WIDE>(src, m), ry = fetch8<WIDE>(src, m + 8);
  if (pos < 0 || pos >= a.max_positions) {
    if (in && hd == 0 && m == 0) report(a.status, NQB200_ERR_BAD_INDEX);
    pos = 0;
  }
  Half x = unpack8<BF16>(rx), y = unpack8<BF16>(ry);
  norm_turn<BF16>(x, y, fetch8<WIDE>(weight, m), fetch8<WIDE>(weight, m + 8), angles_of(a.cos_sin + pos * kDim), a.eps, !is_v);
  if (__any_sync(0xFFFFFFFFu, in && !is_q)) {          // (a warp's other heads go along)
    uint2 words, params;
    quantise<BF16>(x, y, words, params);
    if (in && !is_q) {
      const int64_t row = a.rows[t], page = row >= 0 && row <= INT32_MAX ? (int64_t)((uint32_t)row / (uint32_t)a.cache.block) : row / a.cache.block;
      if (row >= 0 && page < a.cache.pages) {
        const int r = (int)(row - page * a.cache.block);
        uint8_t* base = (is_v ? a.cache.v : a.cache.k) + page_at(a.cache, page, is_v ? hd - Hq - Hkv : hd - Hq);
        reinterpret_cast<uint2*>(base + r * kData)[m] = words;
        if (m == 0) *reinterpret_cast<uint2*>(base + (int64_t)a.cache.block * kData + r * kParams) = params;
      } else if (row >= 0 && m == 0) {
        report(a.status, NQB200_ERR_BAD_INDEX);
      }
    }
  }
  if (in && is_q) {
    uint4* dst = reinterpret_cast<uint4*>(a.q_out + ((int64_t)t * Hq + hd) * kDim);
    dst[m] = pack8<BF16>(x);
    dst[m + 8] = pack8<BF16>(y);
  }
}

// 16 lanes per (row, head of k or v), lane l takes word l: 8 dimensions, 16 bytes out.
template <bool BF16>
__global__ void __launch_bounds__(256) kv4_load_kernel(Cache c, const int64_t* rows, uint16_t* k_out, uint16_t* v_out, int n, int* status) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 15, at = blockIdx.x * 16 + (threadIdx.x >> 4), per = 2 * c.kv_heads;
  if (at >= n * per) return;
  const int i = at / per, hd = at - i * per;
  const bool is_v = hd >= c.kv_heads;
  const int h = is_v ? hd - c.kv_heads : hd;
  const int64_t row = rows[i], page = row / c.block;
  uint32_t out[4] = {0u, 0u, 0u, 0u};
  if (row >= 0 && page < c.pages) {
    const int r = (int)(row - page * c.block);
    const uint8_t* base = (is_v ? c.v : c.k) + page_at(c, page, h);
    const uint32_t word = reinterpret_cast<const uint32_t*>(base + r * kData)[lane];
    const uint32_t p = reinterpret_cast<const uint32_t*>(base + (int64_t)c.block * kData + r * kParams)[lane & 1];
    const float s = scale_of<BF16>(p), m = offset_of<BF16>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      out[e] = (uint32_t)float_to_raw16<BF16>(level<BF16>(nibble(word, e), s, m)) | ((uint32_t)float_to_raw16<BF16>(level<BF16>(nibble(word, e + 4), s, m)) << 16);
  } else if (row >= 0 && lane == 0) {
    report(status, NQB200_ERR_BAD_INDEX);
  }
  uint16_t* dst = (is_v ? v_out : k_out) + ((int64_t)i * c.kv_heads + h) * kDim + (lane & 1) * kGroup + (lane >> 1) * 8;
  *reinterpret_cast<uint4*>(dst) = make_uint4(out[0], out[1], out[2], out[3]);
}

}  // namespace
}  // namespace nqb200

using namespace nqb200;

extern "C" int nqb200_kv4_store(const void* qkv, int64_t row_stride, const void* q_weight, const void* k_weight, const float* cos_sin,
                                int64_t max_positions, const int64_t* positions, const int64_t* rows, const nqb200_kv4* cache, void* q_out, int64_t T,
                                int64_t num_q_heads, float eps, int dtype, int* status, void* stream) {
  const int rc = kv4::check_cache(cache);
  if (rc != NQB200_OK) return rc;
  if (T < 0 || num_q_heads <= 0 || num_q_heads > 65535 || max_positions <= 0 || row_stride < (num_q_heads + 2 * cache->kv_heads) * kv4::kDim || row_stride % 4 != 0)
    return NQB200_ERR_BAD_SHAPE;
  if (dtype != NQB200_F16 && dtype != NQB200_BF16) return NQB200_ERR_BAD_DTYPE;
  if (T == 0) return NQB200_OK;
  if (T > (INT32_MAX - 32) / (num_q_heads + 2 * cache->kv_heads)) return NQB200_ERR_TOO_LARGE;
  if (!qkv || !q_weight || !k_weight || !cos_sin || !positions || !rows || !q_out) return NQB200_ERR_NULL_POINTER;
  const auto on8 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; };
  if (!on8(qkv) || !on8(q_weight) || !on8(k_weight) || !aligned16(q_out) || !aligned16(cos_sin)) return NQB200_ERR_MISALIGNED;
  const bool wide = row_stride % 8 == 0 && aligned16(qkv) && aligned16(q_weight) && aligned16(k_weight);
  StoreArgs a = {(const uint16_t*)qkv, row_stride, (const uint16_t*)q_weight, (const uint16_t*)k_weight, cos_sin, max_positions, positions, rows,
                 kv4::cache_of(cache), (uint16_t*)q_out, (int)T, (int)num_q_heads, eps, status};
  const int64_t heads = T * (num_q_heads + 2 * cache->kv_heads);
  const auto kernel = dtype == NQB200_BF16 ? (wide ? kv4_store_kernel<true, true> : kv4_store_kernel<true, false>) : (wide ? kv4_store_kernel<false, true> : kv4_store_kernel<false, false>);
  return launch_overlapped(kernel, dim3((unsigned)((heads + 31) / 32)), dim3(256), 0,
                           (cudaStream_t)stream, a);
}

extern "C" int nqb200_kv4_load(const nqb200_kv4* cache, const int64_t* rows, void* k_out, void* v_out, int64_t n, int dtype, int* status, void* stream) {
  const int rc = kv4::check_cache(cache);
  if (rc != NQB200_OK) return rc;
  if (n < 0) return NQB200_ERR_BAD_SHAPE;
  if (dtype != NQB200_F16 && dtype != NQB200_BF16) return NQB200_ERR_BAD_DTYPE;
  if (n == 0) return NQB200_OK;
  if (n > (INT32_MAX - 16) / (2 * cache->kv_heads)) return NQB200_ERR_TOO_LARGE;
  if (!rows || !k_out || !v_out) return NQB200_ERR_NULL_POINTER;
  if (!aligned16(k_out) || !aligned16(v_out)) return NQB200_ERR_MISALIGNED;
  return launch_overlapped(dtype == NQB200_BF16 ? kv4_load_kernel<true> : kv4_load_kernel<false>, dim3((unsigned)((n * 2 * cache->kv_heads + 15) / 16)), dim3(256), 0,
                           (cudaStream_t)stream, kv4::cache_of(cache), rows, (uint16_t*)k_out, (uint16_t*)v_out, (int)n, status);
}
