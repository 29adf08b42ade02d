// Attention over the 4-bit key/value cache: one token per sequence (with norm, rotation and store of that token), and several.
//
// A CTA takes a query head of a token; its warps take keys in turn, a lane four dimensions of each, and keep a running maximum and sum.
#include "kv4.cuh"

namespace nqb200 {
namespace {

using namespace kv4;
constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const uint16_t* q; int64_t stride;              // queries, or the projections of a decode step
  const uint16_t *qw, *kw;                        // decode only, as are the next three
  const float* cos_sin; int64_t max_positions;
  const int64_t *positions, *rows;
  Cache cache;
  const int32_t* table; int64_t width;
  const int32_t *ctx, *cu, *pos0;
  uint16_t* out;
  int batch, heads, max_len, max_ctx;
  float scale, eps;
  int* status;
};

// Four dimensions 4 lane .. + 3 of a stored row.
template <bool BF16> __device__ __forceinline__ void fetch(const uint32_t* row, uint2 params, float (&x)[4]) {
  const int lane = threadIdx.x & 31, j = lane >> 4, m = (lane & 15) >> 1, half = lane & 1;
  const uint32_t word = row[2 * m + j], p = j ? params.y : params.x;
  const float s = scale_of<BF16>(p), off = offset_of<BF16>(p);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = fmaf(nibble(word, 2 * half + (e >> 1) + 4 * (e & 1)), s, off);
}

template <bool BF16, bool DECODE>
__global__ void __launch_bounds__(32 * kWarps) kv4_rows_kernel(const __grid_constant__ Args a) {
  __shared__ __align__(16) uint32_t own[2][kData / 4];
  __shared__ uint2 own_params[2];
  __shared__ float s_q[kDim], s_o[kWarps][kDim], s_m[kWarps], s_l[kWarps];
  grid_launch_dependents();
  grid_dependency_wait();
  const int h = blockIdx.x, t = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, R = a.heads / a.cache.kv_heads, kvh = h / R;
  int b = t, keys;
  if (DECODE) {
    keys = a.ctx[t];
  } else {
    int hi = a.batch;                              // cu[b] <= t < cu[b + 1]
    for (b = 0; hi - b > 1;) {
      const int mid = (b + hi) / 2;
      if (a.cu[mid] <= t) b = mid; else hi = mid;
    }
    keys = a.pos0[b] + t - a.cu[b] + 1;
  }
  uint16_t* out = a.out + ((int64_t)t * a.heads + h) * kDim;
  const int64_t room = a.width * a.cache.block;
  if (keys > room) { if (threadIdx.x == 0) report(a.status, NQB200_ERR_BAD_INDEX); keys = (int)room; }
  if (keys <= 0) { out[threadIdx.x] = 0; return; }
  if (DECODE) {
    // half a warp a head: the query, the key, the value
    const int l = threadIdx.x & 15, who = threadIdx.x >> 4;
    const uint16_t* src = a.q + (int64_t)t * a.stride + (int64_t)(who == 0 ? h : who == 1 ? a.heads + kvh : a.heads + a.cache.kv_heads + kvh) * kDim;
    float x[4], y[4], ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = raw16_to_float<BF16>(src[4 * l + e]);
      y[e] = raw16_to_float<BF16>(src[64 + 4 * l + e]);
      ss += x[e] * x[e] + y[e] * y[e];
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
    int64_t pos = a.positions[t];
    if (pos < 0 || pos >= a.max_positions) { if (threadIdx.x == 0) report(a.status, NQB200_ERR_BAD_INDEX); pos = 0; }
    if (who < 2) {
      const float inv = rsqrtf(ss / (float)kDim + a.eps);
      const uint16_t* w = who ? a.kw : a.qw;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float u = x[e] * inv * raw16_to_float<BF16>(w[4 * l + e]), v = y[e] * inv * raw16_to_float<BF16>(w[64 + 4 * l + e]);
        const float c = a.cos_sin[pos * kDim + 4 * l + e], s = a.cos_sin[pos * kDim + 64 + 4 * l + e];
        x[e] = u * c - v * s;
        y[e] = u * s + v * c;
      }
    }
    if (who == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) { s_q[4 * l + e] = x[e]; s_q[64 + 4 * l + e] = y[e]; }
    }
    uint32_t word;
    uint2 params;
    quantise<BF16>(x, y, word, params);
    if (who == 1 || who == 2) {
      own[who - 1][l] = word;
      if (l == 0) own_params[who - 1] = params;
      const int64_t row = a.rows[t], page = row / a.cache.block;
      if (h % R == 0 && row >= 0 && page < a.cache.pages) {
        const int r = (int)(row - page * a.cache.block);
        uint8_t* base = (who == 2 ? a.cache.v : a.cache.k) + page_at(a.cache, page, kvh);
        reinterpret_cast<uint32_t*>(base + r * kData)[l] = word;
        if (l == 0) *reinterpret_cast<uint2*>(base + (int64_t)a.cache.block * kData + r * kParams) = params;
      } else if (row >= 0 && page >= a.cache.pages && l == 0) {
        report(a.status, NQB200_ERR_BAD_INDEX);
      }
    }
  } else {
    s_q[threadIdx.x] = raw16_to_float<BF16>(a.q[(int64_t)t * a.stride + (int64_t)h * kDim + threadIdx.x]);
  }
  __syncthreads();
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, sum = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) q[e] = s_q[4 * lane + e] * (a.scale * kLog2e);
  for (int j = warp; j < keys; j += kWarps) {
    float x[4], v[4];
    if (DECODE && j == keys - 1) {
      fetch<BF16>(own[0], own_params[0], x);
      fetch<BF16>(own[1], own_params[1], v);
    } else {
      const int page = a.table[(int64_t)b * a.width + j / a.cache.block], r = j % a.cache.block;
      if (page < 0 || page >= a.cache.pages) { if (lane == 0) report(a.status, NQB200_ERR_BAD_INDEX); continue; }
      const int64_t at = page_at(a.cache, page, kvh), par = at + (int64_t)a.cache.block * kData + r * kParams;
      fetch<BF16>(reinterpret_cast<const uint32_t*>(a.cache.k + at + r * kData), *reinterpret_cast<const uint2*>(a.cache.k + par), x);
      fetch<BF16>(reinterpret_cast<const uint32_t*>(a.cache.v + at + r * kData), *reinterpret_cast<const uint2*>(a.cache.v + par), v);
    }
    float s = q[0] * x[0] + q[1] * x[1] + q[2] * x[2] + q[3] * x[3];
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, k);
    const float n = max_nan(m, s), f = exp2f(m - n), w = exp2f(s - n);
    sum = sum * f + w;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * f + w * v[e];
    m = n;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) s_o[warp][4 * lane + e] = o[e];
  if (lane == 0) { s_m[warp] = m; s_l[warp] = sum; }
  __syncthreads();
  float top = s_m[0], acc = 0.f, l = 0.f;
  for (int w = 1; w < kWarps; ++w) top = max_nan(top, s_m[w]);
  for (int w = 0; w < kWarps; ++w) {
    const float f = s_m[w] == -INFINITY ? 0.f : exp2f(s_m[w] - top);
    acc += f * s_o[w][threadIdx.x];
    l += f * s_l[w];
  }
  out[threadIdx.x] = float_to_raw16<BF16>(l == 0.f ? 0.f : acc / l);
}

template <bool DECODE> int launch(const Args& a, int64_t tokens, int dtype, cudaStream_t st) {
  return launch_overlapped(dtype == NQB200_BF16 ? kv4_rows_kernel<true, DECODE> : kv4_rows_kernel<false, DECODE>, dim3((unsigned)a.heads, (unsigned)tokens),
                           dim3(32 * kWarps), 0, st, a);
}

}  // namespace
}  // namespace nqb200

using namespace nqb200;

static int check_heads(const nqb200_kv4* cache, int64_t heads, int64_t width, int dtype) {
  const int rc = kv4::check_cache(cache);
  if (rc != NQB200_OK) return rc;
  if (heads <= 0 || heads > 65535 || heads % cache->kv_heads != 0 || width <= 0 || width > INT32_MAX) return NQB200_ERR_BAD_SHAPE;
  return dtype == NQB200_F16 || dtype == NQB200_BF16 ? NQB200_OK : NQB200_ERR_BAD_DTYPE;
}

extern "C" size_t nqb200_kv4_decode_scratch_bytes(int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

extern "C" int nqb200_kv4_decode_attention(const void* qkv, int64_t row_stride, const void* q_weight, const void* k_weight, const float* cos_sin,
                                           int64_t max_positions, const int64_t* positions, const int64_t* rows, const nqb200_kv4* cache,
                                           const int32_t* table, int64_t table_width, const int32_t* ctx, void* out, int64_t batch, int64_t num_q_heads,
                                           float scale, float eps, int dtype, void*, size_t, int* status, void* stream) {
  const int rc = check_heads(cache, num_q_heads, table_width, dtype);
  if (rc != NQB200_OK) return rc;
  if (batch < 0 || batch > 65535 || max_positions <= 0 || row_stride < (num_q_heads + 2 * cache->kv_heads) * kv4::kDim || row_stride % 8 != 0) return NQB200_ERR_BAD_SHAPE;
  if (batch == 0) return NQB200_OK;
  if (!qkv || !q_weight || !k_weight || !cos_sin || !positions || !rows || !table || !ctx || !out) return NQB200_ERR_NULL_POINTER;
  if (!aligned16(qkv) || !aligned16(out)) return NQB200_ERR_MISALIGNED;
  Args a = {};
  a.q = (const uint16_t*)qkv; a.stride = row_stride; a.qw = (const uint16_t*)q_weight; a.kw = (const uint16_t*)k_weight;
  a.cos_sin = cos_sin; a.max_positions = max_positions; a.positions = positions; a.rows = rows; a.cache = kv4::cache_of(cache);
  a.table = table; a.width = table_width; a.ctx = ctx; a.out = (uint16_t*)out; a.batch = (int)batch; a.heads = (int)num_q_heads;
  a.scale = scale; a.eps = eps; a.status = status;
  return launch<true>(a, batch, dtype, (cudaStream_t)stream);
}

extern "C" size_t nqb200_kv4_prompt_scratch_bytes(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

extern "C" int nqb200_kv4_prompt_attention(const void* q, int64_t q_stride, const nqb200_kv4* cache, const int32_t* table, int64_t table_width,
                                           const int32_t* cu, const int32_t* pos0, void* out, int64_t batch, int64_t T, int64_t max_len, int64_t max_ctx,
                                           int64_t tiles, int64_t num_q_heads, float scale, int dtype, void*, size_t, int* status, void* stream) {
  const int rc = check_heads(cache, num_q_heads, table_width, dtype);
  if (rc != NQB200_OK) return rc;
  if (batch < 0 || batch > 65535 || T < 0 || T > 65535 || max_len < 0 || max_ctx < max_len || tiles < 0 || q_stride < num_q_heads * kv4::kDim || q_stride % 8 != 0)
    return NQB200_ERR_BAD_SHAPE;
  if (batch == 0 || T == 0) return NQB200_OK;
  if (!q || !table || !cu || !pos0 || !out) return NQB200_ERR_NULL_POINTER;
  if (!aligned16(q) || !aligned16(out)) return NQB200_ERR_MISALIGNED;
  Args a = {};
  a.q = (const uint16_t*)q; a.stride = q_stride; a.cache = kv4::cache_of(cache); a.table = table; a.width = table_width; a.cu = cu; a.pos0 = pos0;
  a.out = (uint16_t*)out; a.batch = (int)batch; a.heads = (int)num_q_heads; a.max_len = (int)max_len; a.max_ctx = (int)max_ctx; a.scale = scale; a.status = status;
  return launch<false>(a, T, dtype, (cudaStream_t)stream);
}
