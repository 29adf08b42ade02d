// Attention over the 4-bit key/value cache for many queries: prompts and their portions, on the 5th-generation tensor cores.
//
// Two launches.  The first takes the visible pages apart, once, into tiles of 128 keys and 128 values in float16, each 32 KB as the tensor
// cores want it in shared memory (blocks of 64 dimensions, rows of 128 bytes, swizzled), so that the second fetches a tile with one bulk copy
// and needs no tensor map.  float16 whatever the model's type: keys, values and weights in bfloat16 cost twice the error of the
// result's own rounding (a prompt of 8000 tokens: 0.0031 in the 2-norm, 0.0017 so).  A bfloat16 model may have numbers that float16 would not
// hold well.  A tile of keys is then in units of a power of two, and so is a query.  A tile of values has no unit, since weights times units would
// lose what float16 does not hold of the product: it is in bfloat16 instead, and its weights are (values_fit).  So values that a row does not see, or
// gives no weight, cost it no precision.  Keys come from a norm, which keeps them within a few powers of ten of each other; in a tile whose largest is
// beyond 2^15 those below 2^-28 of it are lost.  Rows behind a sequence's end are zeros, and so is a group of a value that is not finite: where the
// first of those stands is noted, and the rows that see it get NaN at the end, and no other (a weight of 0 times NaN would be one).
//
// In the second a CTA takes 256 rows of a key/value head, as two tiles of 128: a row is a query head of a token, the heads of a group beside
// each other, so that the mask cuts as few tiles as it can and short prompts fill a tile.  It walks over tiles of 128 keys, each in two halves of 64.
//   warp 0        copies: two-stage rings of K tiles and of V tiles.
//   warps 1, 2    one lane of each issues tcgen05.mma for a query tile: S = Q K^T of a half (both operands in shared memory)
//                 and O += P V (P in tensor memory, V in shared memory as it lies there: the operand's rows are keys).
//   warp 3        looks for tiles of keys in other units than 1, tiles of values in bfloat16, and values that are not finite.
//   warps 4-19    softmax: four warps for each half of each query tile, a thread per row and half.
// Tensor memory holds S of both tiles (two halves of 64 columns each) and O of both; P overwrites the first half of its own S.  So four
// chains S -> weights -> O += P V -> next S run beside each other.
//
// The weights are 2^(score - m + 8), so that float16 holds them fully down to 2^-22 of a row's largest; none is above 2^15.  m is the largest
// score of the row's first tile and follows the largest score when it falls behind by more than kLag in log2 units; O and the sums are then
// rescaled, which hardly ever happens.  A half finds out by itself that its scores ask for no move, from their largest magnitude; that the
// other half has not moved it learns from what that one hands on, in the order of the products.  The sum that a row is divided by takes the weights in float, before the product's rounding to 16 bits.
//
// One prompt of 8000 tokens, 32 heads over 8: 474 to 493 us, by the GPU (bfloat16; 1.10 PFLOP/s of visible pairs, 0.68 of the measured peak), 463 to
// 473 in float16, 550 back to back under the power cap, of them about 10 for the first launch; 500 tokens behind 12000, 64 heads over 8, 208 (0.96
// PFLOP/s: 128 CTAs on 148 SMs); 1000 tokens 35.  In between the tensor pipe is 54 % busy, the exponentials' pipe 56 %, issue slots 53 %: the chains
// meet at the pipes.  64 tokens take 16 us by themselves (two launches, first bytes, one tile's chain) and 56 to 65 behind 16000, whose tiles
// are written and read again.  4000 tokens 173; with all values in bfloat16 208, with all keys in units 186.
//
// Where the row tiles are fewer than the SMs, the keys are dealt to several CTAs, whose shares a third launch adds.
//
// Every wait is bounded; on expiry NQB200_ERR_WAIT_TIMEOUT goes to the status word, all roles drain and tensor memory is released.
#include "attention_umma.cuh"
#include "kv4.cuh"
#include "kv4_attention.cuh"
#include <type_traits>

namespace nqb200 {
namespace kv4 {
namespace {

using namespace att;

constexpr int kTileKeys = 128, kThreads = 640, kRows = 256;
constexpr uint32_t kTileBytes = kTileKeys * kDim * 2, kBox = kTileKeys * 128;       // of K or V; of a block of 64 dimensions
constexpr uint32_t kColS = 0, kColO = 256, kTmemCols = 512;
constexpr float kLog2e = 1.4426950408889634f, kLag = 7.f, kRoom = 8.f;      // 2^(kLag + kRoom) is a number of float16
constexpr float kLeast = 1e-37f;
constexpr int kNone = 0x7FFFFFFF;

struct alignas(16) TileInfo {
  int bad[2];            // the tile's first key whose value is not finite in dimensions 0..63, in 64..127, or kNone
  float k;               // unit of the tile's keys
  int wide;              // 0: values in float16; else in bfloat16, 1 + the binary orders above kMostOrder of the largest
};
// The unit of numbers up to `top`: 1 where float16 holds them well (its spacing of 2^-24 below 2^-14 is half of a rounding of 2^-12), else the
// power of two that puts `top` between 2^13 and 2^14.
__device__ __forceinline__ float unit_of(float top) {
  if (top == 0.f || (top >= 0.000244140625f && top < 32768.f)) return 1.f;
  const uint32_t e = min(max(__float_as_uint(top) >> 23, 15u), 254u);
  return __uint_as_float((e - 13u) << 23);
}
// Whether float16 products hold values up to `top` in a group as well as others have to be: rounded to float16 they are 2^-13 of the group's largest off
// at most, and a weight that float16 no longer holds (half of its spacing is 2^-33 of the row's largest) takes 2^-21 at most, which is
// 2^-9 of the smallest group's.
__device__ __forceinline__ bool values_fit(float top) { return top == 0.f || (top >= 0.000244140625f && top < 4096.f); }
// Weights times values of more than this many binary orders could leave float's range: such tiles count as higher scores, in the rows' references.
constexpr int kMostOrder = 75;
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool BF16> __device__ __forceinline__ uint32_t pack16(float lo, float hi) { return BF16 ? pack_bf16(lo, hi) : pack_half(lo, hi); }

struct Params {
  const uint16_t* q; int64_t q_stride;
  Cache cache;
  const int32_t* table; int64_t width;
  const int32_t *cu, *pos0;
  uint16_t* out;
  uint8_t* tiles;        // [tile of a sequence][kv head][K, V][kTileBytes]
  TileInfo* info;        // [tile][kv head]
  float* shares;
  int heads, tokens, batch, parts, max_len, max_ctx, total;     // total: tiles that there is room for
  float factor;          // scale log2 e, above 0
  float sign;            // of the scale: the queries take it
  int* status;
};

// Tokens and keys of a sequence, within what the host has said.
struct Span { int first, n, pos0, keys; };
__device__ __forceinline__ Span span_of(const Params& p, int b) {
  Span s;
  s.first = p.cu[b];
  s.n = p.cu[b + 1] - s.first;
  s.pos0 = p.pos0[b];
  if (s.first < 0 || s.n < 0 || s.n > p.max_len || s.n > p.tokens - s.first || s.pos0 < 0) s.n = 0;      // reported by expand
  s.keys = s.n > 0 ? (int)min(min((int64_t)s.pos0 + s.n, (int64_t)p.max_ctx), p.width * p.cache.block) : 0;
  return s;
}
// Tiles of the sequences before b; by all threads of a warp.  Numbers on the device may add up to more than 31 bits where they are not the host's:
// a sum stops above kMostTiles, which no scratch has room for.
__device__ __forceinline__ int tiles_before(const Params& p, int b) {
  int sum = 0;
  for (int i = threadIdx.x & 31; i < b; i += 32) sum = min(sum + (span_of(p, i).keys + kTileKeys - 1) / kTileKeys, 2 * kMostTiles);
  return __reduce_add_sync(0xFFFFFFFFu, sum);
}

// A tile of 128 rows of a key/value head: 16 lanes a row, lane 2 m + j takes word 2 m + j, 8 dimensions, 16 bytes out.
template <bool BF16>
__global__ void __launch_bounds__(512, 3) kv4_expand_kernel(const __grid_constant__ Params p) {
  __shared__ int s_before, s_bad[2], s_unfit;
  __shared__ uint32_t s_top[2];
  grid_launch_dependents();
  grid_dependency_wait();
  const int b = blockIdx.z, h = blockIdx.y, tile = blockIdx.x, lane = threadIdx.x & 15;
  const Span s = span_of(p, b);
  if (tile == 0 && h == 0 && threadIdx.x == 0) {
    const int n = p.cu[b + 1] - p.cu[b];
    if (s.n != n || (n > 0 && s.keys != (int64_t)s.pos0 + n)) report(p.status, NQB200_ERR_BAD_INDEX);
  }
  const int key0 = tile * kTileKeys;
  if (key0 >= s.keys) return;
  if (threadIdx.x < 2) { s_bad[threadIdx.x] = kNone; s_top[threadIdx.x] = 0u; }
  if (threadIdx.x == 0) s_unfit = 0;
  if (threadIdx.x < 32) {
    const int before = tiles_before(p, b);
    if (threadIdx.x == 0) s_before = before;
  }
  __syncthreads();
  const int64_t at = (int64_t)s_before + tile;
  if (at >= p.total) {
    if (threadIdx.x == 0) report(p.status, NQB200_ERR_BAD_INDEX);
    return;
  }
  uint8_t* dst = p.tiles + (at * p.cache.kv_heads + h) * (2 * (int64_t)kTileBytes);
  const int j = lane & 1, m = lane >> 1;
  constexpr int kPer = kTileKeys / 32;          // rows of a thread
  uint32_t word[2][kPer], params[2][kPer];
  bool there[kPer];
  float top[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = i * 32 + (threadIdx.x >> 4), key = key0 + r, blk = key / p.cache.block;
    const int page = key < s.keys ? p.table[(int64_t)b * p.width + blk] : 0;
    there[i] = key < s.keys && page >= 0 && page < p.cache.pages;
    if (key < s.keys && !there[i] && lane == 0) report(p.status, NQB200_ERR_BAD_INDEX);
    const int64_t base = there[i] ? page_at(p.cache, page, h) : 0, row = there[i] ? key - (int64_t)blk * p.cache.block : 0;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const uint8_t* c = (which ? p.cache.v : p.cache.k) + base;
      word[which][i] = reinterpret_cast<const uint32_t*>(c + row * kData)[lane];
      params[which][i] = *reinterpret_cast<const uint32_t*>(c + (int64_t)p.cache.block * kData + row * kParams + 4 * j);
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const float sc = scale_of<BF16>(params[which][i]), off = offset_of<BF16>(params[which][i]), most = max_nan(fabsf(off), fabsf(fmaf(15.f, sc, off)));
      if (there[i] && most < INFINITY) {
        top[which] = fmaxf(top[which], most);
        if (BF16 && which && !values_fit(most)) s_unfit = 1;
      } else if (there[i] && which) {
        atomicMin(&s_bad[j], key0 + i * 32 + (int)(threadIdx.x >> 4));
      }
    }
  }
  if (BF16) {                                   // (float16 holds a float16 model's numbers)
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const uint32_t all = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(top[which]));
      if ((threadIdx.x & 31) == 0) atomicMax(&s_top[which], all);
    }
  }
  __syncthreads();
  const float unit = BF16 ? unit_of(__uint_as_float(s_top[0])) : 1.f, by = 1.f / unit;      // a power of two
  const bool wide = BF16 && s_unfit;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = i * 32 + (threadIdx.x >> 4);
      const float sc = scale_of<BF16>(params[which][i]) * (which ? 1.f : by), off = offset_of<BF16>(params[which][i]) * (which ? 1.f : by);
      const bool zero = !there[i] || (which && !(max_nan(fabsf(off), fabsf(fmaf(15.f, sc, off))) < INFINITY));
      uint32_t out[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lo = nibble(word[which][i], e), hi = nibble(word[which][i], e + 4);
        out[e] = zero ? 0u : BF16 ? pack_half(fmaf(lo, sc, off), fmaf(hi, sc, off)) : pack_half(level<false>(lo, sc, off), level<false>(hi, sc, off));
      }
      if (BF16 && which && wide) {
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = zero ? 0u : pack_bf16(level<true>(nibble(word[1][i], e), sc, off), level<true>(nibble(word[1][i], e + 4), sc, off));
      }
      *reinterpret_cast<uint4*>(dst + which * kTileBytes + j * kBox + r * 128 + ((m ^ (r & 7)) << 4)) = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
  if (threadIdx.x == 0) {
    const int order = (int)(s_top[1] >> 23) - 127;
    p.info[at * p.cache.kv_heads + h] = TileInfo{{s_bad[0], s_bad[1]}, unit, wide ? 1 + max(order + 1 - kMostOrder, 0) : 0};
  }
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

template <bool BF16>
__global__ void __launch_bounds__(kThreads, 1) kv4_prompt_kernel(const __grid_constant__ Params p) {
  constexpr uint32_t kQBytes = 128 * kDim * 2, kOffK = 2 * kQBytes, kOffV = kOffK + 2 * kTileBytes;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_kfull[2], bar_kfree[2], bar_vfull[2], bar_vfree[2], bar_s[2][2], bar_p[2][2], bar_pv[2][2], bar_o[2], bar_x[2][4], bar_m[2][2][4], bar_bad, bar_drain;
  __shared__ float s_x[2][2][2][128], s_m[2][2][128];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort_i, s_before, s_bad[2], s_special;
  __shared__ float s_row[kRows];     // units of the queries
  volatile int* s_abort = &s_abort_i;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem_q = smem_raw + (smem - smem_u32(smem_raw));
  const int warp = warp_index(), lane = threadIdx.x & 31;

  grid_launch_dependents();
  grid_dependency_wait();
  const int b = blockIdx.z, kvh = blockIdx.y, R = p.heads / p.cache.kv_heads;
  const Span sp = span_of(p, b);
  const int rows = sp.n * R, part = blockIdx.x % p.parts;
  const int i0 = (int)(gridDim.x / p.parts - 1 - blockIdx.x / p.parts) * kRows;     // long rows first
  if (i0 >= rows) return;
  // key tiles of this CTA, from `first` on, for each query tile
  const auto pos_of = [&](int row) { return (int)min((int64_t)sp.pos0 + min(row, rows - 1) / R, (int64_t)INT32_MAX); };
  const auto tiles_of = [&](int q) { return i0 + q * 128 < rows ? min(pos_of(i0 + q * 128 + 127), sp.keys - 1) / kTileKeys + 1 : 0; };
  const int all = max(tiles_of(0), tiles_of(1)), per = (all + p.parts - 1) / p.parts, first = part * per;
  int nq[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) nq[q] = __shfl_sync(0xFFFFFFFFu, min(max(tiles_of(q) - first, 0), per), 0);
  const int nmax = max(nq[0], nq[1]), kstart = first * kTileKeys;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&bar_kfull[s]), 1); mbar_init(smem_u32(&bar_kfree[s]), 2);
      mbar_init(smem_u32(&bar_vfull[s]), 1); mbar_init(smem_u32(&bar_vfree[s]), 2);
      mbar_init(smem_u32(&bar_s[s][0]), 1); mbar_init(smem_u32(&bar_s[s][1]), 1); mbar_init(smem_u32(&bar_p[s][0]), 4); mbar_init(smem_u32(&bar_p[s][1]), 4);
      mbar_init(smem_u32(&bar_pv[s][0]), 1); mbar_init(smem_u32(&bar_pv[s][1]), 1); mbar_init(smem_u32(&bar_o[s]), 1);
    }
    for (int s = 0; s < 8; ++s) {
      mbar_init(smem_u32(&bar_x[s >> 2][s & 3]), 2);
      mbar_init(smem_u32(&bar_m[s >> 2][0][s & 3]), 32); mbar_init(smem_u32(&bar_m[s >> 2][1][s & 3]), 32);
    }
    mbar_init(smem_u32(&bar_bad), 1);
    mbar_init(smem_u32(&bar_drain), 2);
    s_abort_i = 0;
    mbar_fence_init();
  }
  if (warp == 1) { tmem_alloc(smem_u32(&s_tmem), kTmemCols); tmem_relinquish(); }
  // A ring stage's first tiles are under way while the queries come in.
  const auto tile_src = [&](int j) { return p.tiles + ((int64_t)(s_before + first + j) * p.cache.kv_heads + kvh) * (2 * (int64_t)kTileBytes); };
  const auto copy = [&](uint32_t dst, const uint8_t* src, uint64_t* bar) {
    mbar_expect_tx(smem_u32(bar), kTileBytes);
    bulk_load(dst, src, kTileBytes, smem_u32(bar));
  };
  if (warp == 0) {
    const int before = tiles_before(p, b);
    if (lane == 0) s_before = before;
    __syncwarp();
    if (before + first + nmax <= p.total && elect_one()) {
      for (int j = 0; j < min(nmax, 2); ++j) {
        copy(smem + kOffK + j * kTileBytes, tile_src(j), &bar_kfull[j]);
        copy(smem + kOffV + j * kTileBytes, tile_src(j) + kTileBytes, &bar_vfull[j]);
      }
    }
  } else {
    // the queries, 16 lanes a row, all of a thread's loads under way at once: block of 64 dimensions, row of 128 bytes, piece swizzled by the row
    constexpr int kWays = kThreads / 16 - 2, kTurns = (kRows + kWays - 1) / kWays;
    const int way = (threadIdx.x >> 4) - 2, l = threadIdx.x & 15;
    uint4 v[kTurns];
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
      const int row = i0 + way + k * kWays;
      v[k] = make_uint4(0u, 0u, 0u, 0u);
      if (way + k * kWays < kRows && row < rows)
        v[k] = reinterpret_cast<const uint4*>(p.q + (int64_t)(sp.first + row / R) * p.q_stride + (int64_t)(kvh * R + row % R) * kDim)[l];
    }
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
      const int i = way + k * kWays;
      float x[8], unit = 1.f;
      values(unpack8<BF16>(v[k]), x);
      if (BF16) {                      // (float16 goes in as it is)
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.f);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        unit = unit_of(top);
      }
      if (i >= kRows) break;           // (the same for a warp's two rows)
      const float by = p.sign / unit;
      if (l == 0) s_row[i] = unit;
      *reinterpret_cast<uint4*>(smem_q + (i >> 7) * kQBytes + (l >> 3) * kBox + (i & 127) * 128 + (((l & 7) ^ (i & 7)) << 4)) =
          make_uint4(pack_half(x[0] * by, x[1] * by), pack_half(x[2] * by, x[3] * by), pack_half(x[4] * by, x[5] * by), pack_half(x[6] * by, x[7] * by));
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // before the tensor cores read them
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int tile0 = s_before + first;                              // of the scratch
  const bool fits = tile0 + nmax <= p.total;                       // (the first launch has reported it)
  if (!fits) nq[0] = nq[1] = 0;
  const int n_tiles = fits ? nmax : 0;

  // of the 96 registers a thread that 640 threads can have: 32 x 128 + 112 x 512 = 96 x 640
  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 32;"); else asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
  if (warp == 0) {
    // --------------------------------------------------------------- copies
    const bool el = elect_one();
    int issued = min(n_tiles, 2);
    for (int j = 2; j < n_tiles; ++j, ++issued) {
      const int s = j & 1;
      if (!wait_bar_warp(&bar_kfree[s], ((j >> 1) - 1) & 1, s_abort, p.status)) break;
      if (el) copy(smem + kOffK + s * kTileBytes, tile_src(j), &bar_kfull[s]);
      if (!wait_bar_warp(&bar_vfree[s], ((j >> 1) - 1) & 1, s_abort, p.status)) {
        mbar_wait(smem_u32(&bar_kfull[s]), (j >> 1) & 1);
        break;
      }
      if (el) copy(smem + kOffV + s * kTileBytes, tile_src(j) + kTileBytes, &bar_vfull[s]);
    }
    // do not leave while a copy may still be landing
    for (int j = issued > 2 ? issued - 2 : 0; j < issued; ++j) {
      mbar_wait(smem_u32(&bar_kfull[j & 1]), (j >> 1) & 1);
      mbar_wait(smem_u32(&bar_vfull[j & 1]), (j >> 1) & 1);
    }
  } else if (warp < 3) {
    // ------------------------------------------------------------------ MMA
    // A warp per query tile, of which one lane issues (elect_one).  A half's S may overwrite its weights once their product has
    // completed.  A ring stage is handed back by both warps, by its only user twice.
    const int q = warp - 1;
    const bool el = elect_one();
    const uint32_t idesc_s = umma_idesc(0, 128, kTileKeys / 2);
    const uint32_t idesc_o = umma_idesc(0, 128, kDim) | (1u << 16), idesc_w = umma_idesc(1, 128, kDim) | (1u << 16);   // B's rows run along k
    const uint64_t dq = umma_smem_desc_sw128(smem + q * kQBytes), dk = umma_smem_desc_sw128(smem + kOffK), dv = smem_desc_mn(smem + kOffV, kBox);
    const uint32_t k_hi = (uint32_t)(dq >> 32), v_hi = (uint32_t)(dv >> 32), q_lo = (uint32_t)dq, k_lo = (uint32_t)dk, v_lo = (uint32_t)dv;
    const uint32_t tS = tmem + kColS + q * 128, tO = tmem + kColO + q * 128;
    const int mine = nq[q], others = nq[q ^ 1];
    bool ok = mine > 0, special = false;
    for (int j = 0; ok && j <= mine; ++j) {
      const int i = j - 1, s = j & 1, so = s ^ 1;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (j > 0) {      // O += P V of the tile before
          if (half == 0) ok = poll_bar_warp(&bar_vfull[so], (i >> 1) & 1, s_abort, p.status);
          ok = ok && poll_bar_warp(&bar_p[q][half], so, s_abort, p.status);
          if (!ok) break;
          tc_fence_after();
          if (BF16 && i == 0) special = s_special;      // (the weights were made behind warp 3's report)
          const bool wide = special && p.info[(int64_t)(tile0 + i) * p.cache.kv_heads + blockIdx.y].wide != 0;
          if (el) {
#pragma unroll
            for (int ks = 0; ks < kTileKeys / 32; ++ks)
              umma_ts_lohi(tO, tS + half * 64 + ks * 8, v_lo + so * (kTileBytes >> 4) + half * (8192 >> 4) + ks * (2048 >> 4), v_hi, wide ? idesc_w : idesc_o,
                           (i > 0 || half > 0 || ks > 0) ? 1u : 0u);
            umma_commit(smem_u32(j == mine && half == 1 ? &bar_o[q] : &bar_pv[q][half]));
            if (half == 1) {
              umma_commit(smem_u32(&bar_vfree[so]));
              if (i >= others) umma_commit(smem_u32(&bar_vfree[so]));
            }
          }
        }
        if (j < mine) {
          if (j > 0) ok = poll_bar_warp(&bar_pv[q][half], so, s_abort, p.status);   // the weights have been read: their place takes the next scores
          if (half == 0) ok = ok && poll_bar_warp(&bar_kfull[s], (j >> 1) & 1, s_abort, p.status);
          if (!ok) break;
          tc_fence_after();
          if (el) {
#pragma unroll
            for (int ks = 0; ks < kDim / 16; ++ks)
              umma_ss_lohi(tS + half * 64, q_lo + (ks >> 2) * (kBox >> 4) + (ks & 3) * 2,
                           k_lo + s * (kTileBytes >> 4) + half * (8192 >> 4) + (ks >> 2) * (kBox >> 4) + (ks & 3) * 2, k_hi, idesc_s, ks > 0 ? 1u : 0u);
            umma_commit(smem_u32(&bar_s[q][half]));
            if (half == 1) {
              umma_commit(smem_u32(&bar_kfree[s]));
              if (j >= others) umma_commit(smem_u32(&bar_kfree[s]));
            }
          }
        }
      }
    }
    // everything issued has completed before tensor memory may be released
    if (el) umma_commit(smem_u32(&bar_drain));
    mbar_wait(smem_u32(&bar_drain), 0);
  } else if (warp == 3) {
    // ------------------------------------------------ units and types of tiles, and values that are not finite
    int low[2] = {kNone, kNone};
    bool special = false;
    for (int j = lane; j < n_tiles; j += 32) {
      const TileInfo v = p.info[(int64_t)(tile0 + j) * p.cache.kv_heads + blockIdx.y];
      low[0] = min(low[0], v.bad[0]);
      low[1] = min(low[1], v.bad[1]);
      special = special || v.k != 1.f || v.wide != 0;
    }
#pragma unroll
    for (int g = 0; g < 2; ++g) low[g] = __reduce_min_sync(0xFFFFFFFFu, low[g]);
    special = __any_sync(0xFFFFFFFFu, special);
    if (lane == 0) {
      s_bad[0] = low[0];
      s_bad[1] = low[1];
      s_special = special;
      mbar_arrive(smem_u32(&bar_bad));
    }
  } else {
    // -------------------------------------------------------------- softmax
    const int q = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(32 * quarter) << 16, tS = tmem + lanes + kColS + q * 128 + half * 64, tO = tmem + lanes + kColO + q * 128;
    const int i = i0 + q * 128 + row, pos = pos_of(i);
    auto done = [&]() {           // this half of the weights is in tensor memory
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_p[q][half]));
    };
    int exchanges = 0;
    auto exchange = [&](float mine, float& other) {   // with the thread that has the row's other half
      const int x = exchanges & 1;
      s_x[q][half][x][row] = mine;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_x[q][quarter]));
      const bool got = wait_bar_warp(&bar_x[q][quarter], x, s_abort, p.status);
      tc_fence_after();
      other = s_x[q][half ^ 1][x][row];
      ++exchanges;
      return got;
    };
    // (above 0 with all units in it, where a masked score stays minus infinity; the scores of queries and keys so small are nothing)
    const float row_factor = BF16 ? fmaxf(p.factor * s_row[q * 128 + row], kLeast) : p.factor;
    float m = -INFINITY;
    uint64_t lsum = pair2(0.f, 0.f);
    // A row's reference goes from half to half in the order of their products: 0 and 1 of the first tile, 0 and 1 of the next, and so on,
    // except in the first tile, where both agree on it.
    auto pass = [&](float mine) {    // (every lane arrives: a branch for one of them costs more)
      s_m[q][half][row] = mine;
      mbar_arrive(smem_u32(&bar_m[q][half][quarter]));
    };
    auto take = [&](int n) {       // what the other half passed on, its n-th
      if (!wait_bar_warp(&bar_m[q][half ^ 1][quarter], (n - 1) & 1, s_abort, p.status)) return false;
      const float got = s_m[q][half ^ 1][row];
      if (__any_sync(0xFFFFFFFFu, got != m)) {
        const float f = got != m ? ex2(m - got) : 1.f;
        lsum = mul2(lsum, pair2(f, f));
        m = got;
      }
      return true;
    };
    auto catch_up = [&](int j) {   // with what came before this half of tile j
      if (half == 1) return j == 0 || take(j);
      return j < 2 || take(j - 1);
    };
    bool ok = wait_bar_warp(&bar_bad, 0, s_abort, p.status);
    const int wfirst = pos_of(i - lane);        // the first position of the warp
    // SPECIAL: some tile has keys in units other than 1 or values in bfloat16
    const auto tiles = [&](auto special) {
      constexpr bool SPECIAL = decltype(special)::value;
      for (int j = 0; ok && j < nq[q]; ++j) {
        const bool joint = j == 0;
        ok = catch_up(j) && wait_bar_warp(&bar_s[q][half], j & 1, s_abort, p.status);
        if (!ok) break;
        tc_fence_after();
        const int key0 = kstart + j * kTileKeys + half * 64;
        const bool masked = key0 + 63 > wfirst;     // for any row of the warp
        float factor = row_factor;
        int wide = 0;
        if (SPECIAL) {
          const TileInfo t = p.info[(int64_t)(tile0 + j) * p.cache.kv_heads + blockIdx.y];
          factor = fmaxf(factor * t.k, kLeast);
          wide = t.wide;
        }
        uint32_t r[2][32];     // the row's scores, all of this half
  #pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld32(tS + c * 32, r[c]);
        tc_wait_ld();
        // what the row does not see: scores below all others
        const int left = pos - key0;
        auto mask = [&](uint32_t (&v)[32], int from) {
  #pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = from + e <= left ? v[e] : 0xFF800000u;
        };
        float mx = -INFINITY;  // where it is asked for, the largest score
        bool look = joint || masked;
        if (masked) {
          mask(r[0], 0);
          mask(r[1], 32);
        } else if (!joint) {   // a half finds out from the largest magnitude that nothing moves
          float hi[4] = {0.f, 0.f, 0.f, 0.f};
  #pragma unroll
          for (int c = 0; c < 2; ++c)
  #pragma unroll
            for (int e = 0; e < 32; e += 2) hi[(e >> 1) & 3] = max3_abs(hi[(e >> 1) & 3], __uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1]));
          look = (SPECIAL && wide > 1) || !__all_sync(0xFFFFFFFFu, fmaxf(fmaxf(hi[0], hi[1]), fmaxf(hi[2], hi[3])) * factor <= m + kLag);
        }
        const float lag = m + kLag;
        if (look) {
          float hi[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  #pragma unroll
          for (int c = 0; c < 2; ++c)
  #pragma unroll
            for (int e = 0; e < 32; e += 2) hi[(e >> 1) & 3] = max3(hi[(e >> 1) & 3], __uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1]));
          mx = fmaxf(fmaxf(hi[0], hi[1]), fmaxf(hi[2], hi[3]));
          if (joint) {
            float mo;
            if (!(ok = exchange(mx, mo))) break;
            mx = fmaxf(mx, mo);
          }
          mx = mx == -INFINITY ? mx : mx * factor;
          if (SPECIAL && wide > 1) mx += (float)(wide - 1);
        }
        const bool move = mx > lag;      // also from -inf
        if (!joint) pass(move ? mx : m);
        if (j == 0) {
          m = mx;
        } else if (__any_sync(0xFFFFFFFFu, move)) {
          const float f = move ? ex2(m - mx) : 1.f;
          lsum = mul2(lsum, pair2(f, f));
          m = move ? mx : m;
          // O has the products of all halves before this one, and no other until this one's weights are reported
          if (!(ok = wait_bar_warp(&bar_pv[q][half ^ 1], (j - 1 + half) & 1, s_abort, p.status))) break;
          tc_fence_after();
  #pragma unroll 1
          for (int c = 0; c < kDim / 32; ++c) {
            tmem_ld32(tO + c * 32, r[0]);
            tc_wait_ld();
  #pragma unroll
            for (int e = 0; e < 32; ++e) r[0][e] = __float_as_uint(__uint_as_float(r[0][e]) * f);
            tmem_st32(tO + c * 32, r[0]);
          }
          tc_wait_st();
          tmem_ld32(tS, r[0]);      // the scores again
          tc_wait_ld();
          if (masked) mask(r[0], 0);
        }
        const float mu = (m == -INFINITY ? 0.f : m) - kRoom;
        const uint64_t nm2 = pair2(-mu, -mu), k1 = pair2(factor, factor);
        if (!SPECIAL || wide == 0) {
          uint64_t ls[2] = {lsum, 0};
  #pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t w[16];
  #pragma unroll
            for (int e = 0; e < 16; ++e) {
              float x0, x1;
              unpair2(fma2(pair2(__uint_as_float(r[c][2 * e]), __uint_as_float(r[c][2 * e + 1])), k1, nm2), x0, x1);
              x0 = ex2(x0);
              x1 = ex2(x1);
              w[e] = pack_half(x0, x1);
              ls[e & 1] = add2(ls[e & 1], pair2(x0, x1));
            }
            tmem_st16(tS + c * 16, w);
          }
          lsum = add2(ls[0], ls[1]);
        } else {
          // from tensor memory again, a piece at a time: compact code for tiles whose values are in bfloat16
  #pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t v[16], w[8];
            tmem_ld_32x32b_x16(tS + c * 16, v);
            tc_wait_ld();
  #pragma unroll
            for (int e = 0; e < 8; ++e) {
              float x[2];
  #pragma unroll
              for (int u = 0; u < 2; ++u) x[u] = key0 + c * 16 + 2 * e + u <= pos ? ex2(fmaf(__uint_as_float(v[2 * e + u]), factor, -mu)) : 0.f;
              w[e] = pack_bf16(x[0], x[1]);
              lsum = add2(lsum, pair2(x[0], x[1]));
            }
            tmem_st8(tS + c * 8, w);      // lies behind what has been read of S
          }
        }
        done();
      }
    };
    if (!BF16 || !s_special) tiles(std::false_type()); else tiles(std::true_type());
    // Rows go out through shared memory (the queries' place, which no product reads any more), so that a store's lanes write to four lines and
    // not to 32: a warp stages its 32 rows x 128 bytes, piece c of row r at c ^ r mod 8.
    const int R = p.heads / p.cache.kv_heads, at = min(i, span_of(p, blockIdx.z).n * R - 1);      // (again, rather than in registers until here)
    const int out_row = at == i ? (p.cu[blockIdx.z] + at / R) * p.heads + (int)blockIdx.y * R + at % R : -1;
    const bool shares = p.parts > 1;
    uint8_t* stage = smem_q + q * kQBytes + (half * 4 + quarter) * 4096;
    const auto put = [&](int c, uint4 v) { *reinterpret_cast<uint4*>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) = v; };
    const auto write = [&](uint8_t* base, int64_t row_bytes, int64_t offset) {
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int r = k * 4 + (lane >> 3), to = __shfl_sync(0xFFFFFFFFu, out_row, r);
        const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
        if (to >= 0) *reinterpret_cast<uint4*>(base + to * row_bytes + offset + (lane & 7) * 16) = v;
      }
      __syncwarp();
    };
    float* const share0 = p.shares + (blockIdx.x % p.parts) * kShare;
    const int64_t share_row = (int64_t)p.parts * kShare * sizeof(float);
    if (ok && nq[q] > 0) {
      ok = (half == 1 || catch_up(nq[q])) && wait_bar_warp(&bar_o[q], 0, s_abort, p.status);
      float l = 0.f;
      if (ok) {
        float a, c2, other;
        unpair2(lsum, a, c2);
        l = a + c2;
        ok = exchange(l, other);
        l += other;
      }
      if (ok) {
        tc_fence_after();
        // dimensions 64 half ..: NaN where a value that the row sees is none
        const float poison = s_bad[half] <= pos ? __int_as_float(0x7FC00000) : 0.f;
        const float f = shares ? 1.f : 1.f / l;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t r[32];
          tmem_ld32(tO + half * 64 + c * 32, r);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(fmaf(__uint_as_float(r[e]), f, poison));
          if (shares) {
#pragma unroll
            for (int e = 0; e < 8; ++e) put(e, make_uint4(r[4 * e], r[4 * e + 1], r[4 * e + 2], r[4 * e + 3]));
            write((uint8_t*)share0, share_row, half * 256 + c * 128);
          } else {
            const auto two = [&](int e) { return pack16<BF16>(__uint_as_float(r[e]), __uint_as_float(r[e + 1])); };
#pragma unroll
            for (int e = 0; e < 4; ++e) put(4 * c + e, make_uint4(two(8 * e), two(8 * e + 2), two(8 * e + 4), two(8 * e + 6)));
          }
        }
        if (!shares) write((uint8_t*)p.out, kDim * 2, half * 128);
        if (shares && out_row >= 0 && half == 0) { share0[(int64_t)out_row * p.parts * kShare + kDim] = m; share0[(int64_t)out_row * p.parts * kShare + kDim + 1] = l; }
        tc_fence_before();
      }
    } else if (nq[q] == 0) {      // no keys of this part, or none that could be read
#pragma unroll
      for (int e = 0; e < 8; ++e) put(e, make_uint4(0u, 0u, 0u, 0u));
      if (shares) {
        write((uint8_t*)share0, share_row, half * 256);
        write((uint8_t*)share0, share_row, half * 256 + 128);
        if (out_row >= 0 && half == 0) { share0[(int64_t)out_row * p.parts * kShare + kDim] = -INFINITY; share0[(int64_t)out_row * p.parts * kShare + kDim + 1] = 0.f; }
      } else {
        write((uint8_t*)p.out, kDim * 2, half * 128);
      }
    }
  }
  // all roles meet here, also after a give-up, so that tensor memory is always released
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { __syncwarp(); tc_fence_after(); tmem_dealloc(tmem, kTmemCols); }
}

int64_t tile_bytes(int64_t tiles, int64_t kv_heads) { return tiles * kv_heads * 2 * (int64_t)kTileBytes; }
int64_t info_bytes(int64_t tiles, int64_t kv_heads) { return tiles * kv_heads * (int64_t)sizeof(TileInfo); }

// CTAs that a row tile's keys are dealt to: as many as fill the SMs, with at least four tiles of keys each.
int parts_of(int64_t batch, int64_t max_len, int64_t max_ctx, int64_t heads, int64_t kv_heads) {
  const int64_t ctas = (max_len * (heads / kv_heads) + kRows - 1) / kRows * kv_heads * batch, tiles = (max_ctx + kTileKeys - 1) / kTileKeys;
  int64_t parts = kNumSMs / (ctas > 0 ? ctas : 1);
  if (parts > tiles / 4) parts = tiles / 4;
  return (int)(parts < 1 ? 1 : parts > 64 ? 64 : parts);
}

}  // namespace

// Which of the two ways a call takes: the one that is expected to end first, in us, by what 68 calls of either took (16 to 512 tokens of 1 to 32
// sequences behind 0 to 16000, 2 to 8 query heads per key/value head, 1 and 8 of those; a wrong choice costs 2 us, and up to 10 for
// long drafts of one key/value head).  Few rows: a CTA per 8 of them goes over the keys.  Many: the pages taken apart, then tiles of
// 256 rows x 128 keys one after the other.  64 tokens of 32 heads over 8: 7.2 and 16.2 us alone, 27 and 31 behind 2000, 148 and 56 behind 16000.
bool prompt_umma_faster(int64_t batch, int64_t tokens, int64_t max_len, int64_t max_ctx, int64_t tiles, int64_t heads, int64_t kv_heads) {
  const double rows = (double)tokens * (heads / kv_heads), mean_keys = fmax(1.0, 128.0 * tiles / batch - 0.5 * tokens / batch);
  const double units = (rows / 8 + 0.5 * batch) * kv_heads, few = 5.0 + units * 0.010 + units * mean_keys / 30000;
  const int64_t key_tiles = (max_ctx + kTileKeys - 1) / kTileKeys, parts = parts_of(batch, max_len, max_ctx, heads, kv_heads);
  const double ctas = fmax(rows / kRows, (double)batch) * kv_heads * parts, turns = ctas > kNumSMs ? ctas / kNumSMs : 1.0;
  const bool fresh = max_ctx < 2 * max_len;      // half of the tiles lie behind the mask
  const double many = 12.0 + (max_len * (heads / kv_heads) > 128 ? 2.8 : 0.0) + 0.017 * tiles * kv_heads +
                      2.2 * turns * ((key_tiles + parts - 1) / parts) * (fresh && key_tiles > 2 ? 0.55 : 1.0) + (parts > 1 ? 3.0 : 0.0);
  return many < few;
}
size_t prompt_umma_scratch_bytes(int64_t batch, int64_t tokens, int64_t max_len, int64_t max_ctx, int64_t tiles, int64_t heads, int64_t kv_heads) {
  const int parts = parts_of(batch, max_len, max_ctx, heads, kv_heads);
  return (size_t)(tile_bytes(tiles, kv_heads) + info_bytes(tiles, kv_heads) + (parts > 1 ? tokens * heads * parts * kShare * (int64_t)sizeof(float) : 0));
}
int prompt_umma(const uint16_t* q, int64_t q_stride, const nqb200_kv4* cache, const int32_t* table, int64_t width, const int32_t* cu, const int32_t* pos0,
                uint16_t* out, int64_t batch, int64_t tokens, int64_t max_len, int64_t max_ctx, int64_t tiles, int64_t heads, float scale, int dtype, void* scratch,
                int* status, cudaStream_t st) {
  Params p = {};
  const int64_t hk = cache->kv_heads;
  p.q = q; p.q_stride = q_stride; p.cache = cache_of(cache); p.table = table; p.width = width; p.cu = cu; p.pos0 = pos0; p.out = out;
  p.tiles = (uint8_t*)scratch; p.info = (TileInfo*)(p.tiles + tile_bytes(tiles, hk)); p.shares = (float*)((uint8_t*)p.info + info_bytes(tiles, hk));
  p.heads = (int)heads; p.tokens = (int)tokens; p.batch = (int)batch; p.max_len = (int)max_len; p.max_ctx = (int)max_ctx; p.total = (int)tiles;
  p.parts = parts_of(batch, max_len, max_ctx, heads, hk);
  p.factor = fmaxf(fabsf(scale) * kLog2e, kLeast); p.sign = scale < 0.f ? -1.f : 1.f; p.status = status;
  const bool bf16 = dtype == NQB200_BF16;
  const dim3 expand((unsigned)((max_ctx + kTileKeys - 1) / kTileKeys), (unsigned)hk, (unsigned)batch);
  int rc = launch_overlapped(bf16 ? kv4_expand_kernel<true> : kv4_expand_kernel<false>, expand, dim3(512), 0, st, p);
  if (rc != NQB200_OK) return rc;
  const auto kernel = bf16 ? kv4_prompt_kernel<true> : kv4_prompt_kernel<false>;
  constexpr int smem = 2 * 128 * kDim * 2 + 4 * (int)kTileBytes + 1024;       // one CTA per SM, because a CTA takes all of its tensor memory
  if (!(bf16 ? allow_smem<kv4_prompt_kernel<true>>(smem) : allow_smem<kv4_prompt_kernel<false>>(smem))) return NQB200_ERR_LAUNCH;
  const dim3 grid((unsigned)((max_len * (heads / hk) + kRows - 1) / kRows * p.parts), (unsigned)hk, (unsigned)batch);
  rc = launch_overlapped(kernel, grid, dim3(kThreads), smem, st, p);
  if (rc != NQB200_OK || p.parts == 1) return rc;
  return add_shares(p.shares, out, tokens * heads, p.parts, bf16, st);
}

}  // namespace kv4
}  // namespace nqb200
