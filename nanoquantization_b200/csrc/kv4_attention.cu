// Attention over the 4-bit key/value cache for few queries: one token per sequence, with its norm, rotation and store in the same
// launch, and a few tokens per sequence (drafts, ends of prompts).
//
// Bound by reading the visible keys and values once (144 bytes per key and head) and, next to it, by the instructions that take
// nibbles apart.  A CTA takes up to eight columns of a key/value head (query heads of a token, or of several tokens) and a share of the keys; its warps
// take tiles of 32 keys on their own, through rings that they fill with cp.async.  Both products are mma m16n8k16 with the columns as the
// eight columns of its result:
//
//   numbers  a nibble n becomes 1024 + n or 1024 + 16 n, a pair of them by one logical operation: it goes into the mantissa of float16's
//            1024, one shift for a word of eight.  float16 operands and float accumulators serve both types.
//   scores   per group of 64 dimensions the product of these numbers and the query (which has the sixteenths in it), whose accumulator starts
//            at minus 1024 times the query's sum; score = f (s0 c0 + s1 c1) + m0 q0 + m1 q1 with the key's scales and offsets and the
//            sums of the query's halves, in float.  Keys are exact; the query is rounded to float16 relative to its largest element, a
//            power of two of its own.
//   values   n - 8 by a packed operation more: over thousands of keys a sum with 1024 in it loses what the tensor cores cut off it (1500 keys:
//            0.0022 off), and so does, less, one of numbers above 0.  The weight times the value's scale goes into the product, a version for each
//            of the two groups, rounded to float16 once; a column's products are relative to the largest that it has had, a power of two, so that what
//            is small in float16 is small beside that, in any type.  (Relative to the largest scale alone, a key of large values and no weight
//            took the others' bits.)  What the level 8 stands for is summed in float.
//   order    a lane owns 16 neighbouring bytes of a key and 8 of a value, which one load fetches; which dimension is which row of a
//            product follows from that, as the layout of a row was chosen.
//
// Scores come out relative to a reference, which moves only when one is 8 (in log2 units) above it, found by one vote per 32 keys.  The warps meet in
// shared memory, the CTAs of a cluster in distributed shared memory, several clusters of one sequence in a second launch; always in the same order.
//
// 64 sequences of 3500 keys on average, 64 heads over 8, bfloat16 (263 MB, 40 us at the copy rate): 73 us; float16 81; 45 of 1250, 32 heads over 8 (69
// MB, 10.6 us) 26.4; one of 32000 17.8; one of 37 6.4.  The bytes come in at 3.6 TB/s at most: issue slots are 58 % busy (671 warp
// instructions for 32 keys, of them about 200 to take nibbles and parameters apart, 107 float arithmetic, 64 packed half, 32 products), the ALU
// 51 %, the tensor pipe 22 %, DRAM 40 %, and CTAs of unequal sequences end at different times (IPC 2.3 while they run, 1.9 over all).
#include <cooperative_groups.h>
#include <type_traits>
#include "kv4_attention.cuh"

namespace nqb200 {
namespace {

using namespace kv4;
namespace cg = cooperative_groups;

constexpr int kWarps = 4, kThreads = 32 * kWarps, kTile = 32, kCols = 8;
constexpr int kStage = kTile * 2 * kToken;                    // keys, values, parameters of keys, parameters of values
constexpr int kOffV = kTile * kData, kOffKP = 2 * kTile * kData, kOffVP = kOffKP + kTile * kParams;
constexpr int kOS = kDim + 4;                                 // floats of a column's partial sums
constexpr float kLog2e = 1.4426950408889634f, kLag = 8.f, kAhead = 64.f;      // 2^kLag kAhead is a number of float16

struct Args {
  const uint16_t* q; int64_t stride;              // queries, or the projections of a decode step
  const uint16_t *qw, *kw;                        // decode only, as are the next three
  const float* cos_sin; int64_t max_positions;
  const int64_t *positions, *rows;
  Cache cache;
  const int32_t* table; int width, shift;         // shift: log2 of the block size, or -1
  const int32_t *ctx;                             // decode
  const int32_t *cu, *pos0;                       // several tokens per sequence
  uint16_t* out;
  int heads, groups, tokens, max_len, max_ctx;    // groups: of kCols columns, per key/value head
  float scale, eps;
  float* shares; int parts;                       // a sequence over several clusters (parts > 1): their shares
  int* status;
};

struct Fixed {                                    // behind the rings
  alignas(16) uint16_t q[kCols][kDim + 8];
  alignas(16) uint16_t rest[kCols][kDim + 8];     // what q's rounding left (kRest)
  alignas(16) uint32_t own[2][kData / 4];         // the step's own key and value, as stored
  uint2 own_params[2];
  float m[kWarps][kCols], l[kWarps][kCols];
  float cm[kCols], cl[kCols];                     // of the CTA, read by the cluster
  float unit[kCols];                              // of the queries
  float out[kCols][kDim];
};
__host__ __device__ constexpr int ring_bytes(int stages) { return kWarps * stages * kStage; }
constexpr int smem_bytes(int stages) { return ring_bytes(stages) + (int)sizeof(Fixed); }

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {      // zeros behind `bytes`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes));
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_from(float (&d)[4], const float (&c)[2], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

__device__ __forceinline__ float power_of_two(int n) { return __uint_as_float((uint32_t)(n + 127) << 23); }
__device__ __forceinline__ float max3(float a, float b, float c) { float r; asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }

// Nibbles I and I + 4 of a word, as pairs of float16: 1024 + n for even I, 1024 + 16 n for odd I.  `magic` is a pair of 1024 in a register:
// with two immediate operands it would be two instructions.
struct Lifted { uint32_t v[4]; };
__device__ __forceinline__ Lifted lift(uint32_t w, uint32_t magic) {
  const uint32_t x = w >> 8;
  Lifted r;
  asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(r.v[0]) : "r"(w), "r"(magic));
  asm("lop3.b32 %0, %1, 0x00F000F0, %2, 0xEA;" : "=r"(r.v[1]) : "r"(w), "r"(magic));
  asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(r.v[2]) : "r"(x), "r"(magic));
  asm("lop3.b32 %0, %1, 0x00F000F0, %2, 0xEA;" : "=r"(r.v[3]) : "r"(x), "r"(magic));
  return r;
}
// The same as n - 8.
__device__ __forceinline__ Lifted levels(uint32_t w, uint32_t magic) {
  Lifted r = lift(w, magic);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    __half2& v = *reinterpret_cast<__half2*>(&r.v[i]);
    v = i & 1 ? __hfma2(v, __float2half2_rn(0.0625f), __float2half2_rn(-72.f)) : __hadd2(v, __float2half2_rn(-1032.f));
  }
  return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// A query as the first product's second operand, in units of a power of two that puts its largest element between 256 and 512: eight
// lanes, as in kv4.cuh; elements that meet 1024 + 16 n are divided by 16.  `rest`: what the rounding left.  Returns the unit.
__device__ __forceinline__ float operand(const Half& hx, const Half& hy, uint4& lo, uint4& hi, uint4& lo_rest, uint4& hi_rest) {
  float x[8], y[8], top = 0.f;
  values(hx, x);
  values(hy, y);
#pragma unroll
  for (int e = 0; e < 8; ++e) top = fmaxf(top, fmaxf(fabsf(x[e]), fabsf(y[e])));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  const uint32_t e = min(max(__float_as_uint(top) >> 23, 9u), 253u);
  const float f = __uint_as_float((262u - e) << 23), f16 = f * 0.0625f;
  const auto round = [&](float a, float b, float by, uint32_t& q, uint32_t& left) {
    q = pack2(a * by, b * by);
    const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&q));
    left = pack2(a * by - r.x, b * by - r.y);
  };
  round(x[0], x[1], f, lo.x, lo_rest.x); round(x[2], x[3], f16, lo.y, lo_rest.y); round(x[4], x[5], f, lo.z, lo_rest.z); round(x[6], x[7], f16, lo.w, lo_rest.w);
  round(y[0], y[1], f, hi.x, hi_rest.x); round(y[2], y[3], f16, hi.y, hi_rest.y); round(y[4], y[5], f, hi.z, hi_rest.z); round(y[6], y[7], f16, hi.w, hi_rest.w);
  return __uint_as_float((e - 8u) << 23);
}

// CTAS: of an SM (see split()); they share its registers and its room for rings.  DECODE: one token per sequence whose own key and value are made here.
__host__ __device__ constexpr int stages_of(int ctas) { return ctas == 4 ? 2 : ctas == 3 ? 3 : 4; }
template <bool BF16, bool DECODE, int CTAS>
__global__ void __launch_bounds__(kThreads, CTAS) kv4_rows_kernel(const __grid_constant__ Args a) {
  constexpr int STAGES = stages_of(CTAS);
  constexpr int kRing = ring_bytes(STAGES);
  // A query of a float16 model that comes from float goes in as two numbers: its rounding is half of the error otherwise (3500 keys: 4.1e-4 in
  // the 2-norm with one, 3.0e-4 with two, 2.1e-4 of them the result's own rounding), for 8 % of the time.  Given queries are exact, and
  // bfloat16's results are coarser.
  constexpr bool kRest = DECODE && !BF16;
  extern __shared__ __align__(128) uint8_t smem[];
  Fixed& fx = *reinterpret_cast<Fixed*>(smem + kRing);
  grid_launch_dependents();
  grid_dependency_wait();
  cg::cluster_group cl = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), csize = gridDim.x / a.parts, rank = blockIdx.x % csize;
  const int kvh = blockIdx.y / a.groups, group = blockIdx.y % a.groups, b = blockIdx.z;
  const int R = a.heads / a.cache.kv_heads;
  const int t_first = DECODE ? b : a.cu[b], n_tokens = DECODE ? 1 : a.cu[b + 1] - t_first;
  if (!DECODE && n_tokens != 0 && (t_first < 0 || n_tokens < 0 || n_tokens > a.tokens - t_first)) {      // not rows of q
    if (tid == 0) report(a.status, NQB200_ERR_BAD_INDEX);
    return;
  }
  const int cols = min(kCols, n_tokens * R - group * kCols);     // of this CTA
  if (cols <= 0) return;                                         // the same for the whole cluster
  const int first_pos = DECODE ? 0 : a.pos0[b];
  // column c: row group * 8 + c of the sequence's (token, head of the group) rows
  const auto token_of = [&](int c) { return (group * kCols + c) / R; };
  int keys = DECODE ? a.ctx[b] : (int)min((int64_t)first_pos + token_of(cols - 1) + 1, (int64_t)INT32_MAX);
  const int64_t room = (int64_t)a.width * a.cache.block;
  if (keys > room || (!DECODE && (first_pos < 0 || n_tokens > a.max_len || keys > a.max_ctx))) {
    if (tid == 0) report(a.status, NQB200_ERR_BAD_INDEX);
    keys = (int)min((int64_t)keys, room);
  }
  const int tiles = keys <= 0 ? 0 : (keys + kTile - 1) / kTile, per = (tiles + (int)gridDim.x - 1) / (int)gridDim.x;
  const int t0 = min((int)blockIdx.x * per, tiles), t1 = min(t0 + per, tiles);
  const int stored = DECODE ? keys - 1 : keys;                   // keys that are read from the cache
  const bool newest = DECODE && t1 == tiles && t0 < t1;          // this CTA has the tile with the step's own key
  uint8_t* ring = smem + warp * (STAGES * kStage);
  const uint32_t ring_a = smem_addr(ring);
  const int32_t* table = a.table + (int64_t)b * a.width;

  // 16-byte piece c of row r at r * 64 + (c ^ 2 bit 2 of r) * 16: eight lanes' pieces lie in different banks for keys (two rows that differ
  // in their last bit) and for values (four rows, two of each parity, of which two have bit 2 set).  A copy takes eight rows at a time.
  const int l16 = lane & 15;
  const uint32_t dst_data = ring_a + (lane >> 2) * kData + (((lane & 3) ^ ((lane >> 3) & 2)) << 4), dst_par = ring_a + (lane < 16 ? kOffKP : kOffVP) + l16 * 16;
  const uint8_t* const par_of = (lane < 16 ? a.cache.k : a.cache.v) + (int64_t)a.cache.block * kData;
  const auto page_of = [&](int key, int& row) {
    const int at = a.shift >= 0 ? key >> a.shift : (int)((unsigned)key / (unsigned)a.cache.block);
    row = key - at * a.cache.block;
    return __shfl_sync(0xFFFFFFFFu, table[at], 0);
  };
  auto load = [&](int t, int stage) {
    if (t < t1) {
      const int p0 = t * kTile;
      const uint32_t dst = dst_data + stage * kStage, par = dst_par + stage * kStage;
      int row0;
      const int page = page_of(p0, row0);
      const bool whole = p0 + kTile <= stored && (unsigned)page < (unsigned)a.cache.pages;
      // a whole tile of one page, a whole tile of two pages (16 rows lie in one), and any other: 64 sequences of 4000 keys of 8 heads, us,
      // by the first way, the second and the third: pages of 256 tokens 73.6, 77.0, 85.6; of 16 tokens -, 79.2, 87.8
      int row1 = 0, page1 = -1;
      if (whole && a.cache.block % kTile != 0) page1 = page_of(p0 + 16, row1);
      if (whole && a.cache.block % kTile == 0) {
        const int64_t base = page_at(a.cache, page, kvh);
        const uint8_t *k = a.cache.k + base + row0 * kData + lane * 16, *v = a.cache.v + base + row0 * kData + lane * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          copy16(dst + i * 8 * kData, k + i * 8 * kData, 16);
          copy16(dst + i * 8 * kData + kOffV, v + i * 8 * kData, 16);
        }
        copy16(par, par_of + base + (row0 + 2 * l16) * kParams, 16);
      } else if ((unsigned)page1 < (unsigned)a.cache.pages) {
        const int64_t base0 = page_at(a.cache, page, kvh), base1 = page_at(a.cache, page1, kvh);
        const int64_t at0 = base0 + row0 * kData + lane * 16, at1 = base1 + row1 * kData + lane * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t at = (i < 2 ? at0 : at1) + (i & 1) * 8 * kData;
          copy16(dst + i * 8 * kData, a.cache.k + at, 16);
          copy16(dst + i * 8 * kData + kOffV, a.cache.v + at, 16);
        }
        copy16(par, par_of + (l16 < 8 ? base0 : base1) + ((l16 < 8 ? row0 : row1) + 2 * (l16 & 7)) * kParams, 16);
      } else {
        int64_t base[2];
        int row[2];
        bool there[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = p0 + 16 * h;
          there[h] = key < stored;
          const int pg = there[h] ? page_of(key, row[h]) : 0;
          if (pg < 0 || pg >= a.cache.pages) { there[h] = false; if (lane == 0) report(a.status, NQB200_ERR_BAD_INDEX); }
          base[h] = there[h] ? page_at(a.cache, pg, kvh) : 0;
          if (!there[h]) row[h] = 0;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int h = i >> 1, r = i * 8 + (lane >> 2), bytes = there[h] && p0 + r < stored ? 16 : 0;
          const int64_t src = bytes ? base[h] + (row[h] + (r & 15)) * kData + (lane & 3) * 16 : 0;
          copy16(dst + i * 8 * kData, a.cache.k + src, bytes);
          copy16(dst + i * 8 * kData + kOffV, a.cache.v + src, bytes);
        }
        // parameters of rows 2 l16 and 2 l16 + 1
        const int left = (l16 < 8 ? there[0] : there[1]) ? stored - (p0 + 2 * l16) : 0, bytes = left >= 2 ? 16 : left == 1 ? 8 : 0;
        copy16(par, par_of + (bytes ? (l16 < 8 ? base[0] : base[1]) + ((l16 < 8 ? row[0] : row[1]) + 2 * (l16 & 7)) * kParams : 0), bytes);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int s = 0; s < STAGES - 1; ++s) load(t0 + warp + s * kWarps, s);

  // queries into fx.q, eight lanes each: the first two warps; the step's own key and value: the third
  const int unit = tid >> 3, m8 = tid & 7;
  if (keys > 0 && (warp < 2 || (newest && warp == 2))) {
    const int c = min(unit, cols - 1), idx = group * kCols + c;      // (columns beyond `cols` repeat the last one and are not used)
    const bool is_v = unit == 9;
    const uint16_t* src = DECODE ? a.q + (int64_t)b * a.stride + (int64_t)(warp < 2 ? kvh * R + idx : a.heads + (is_v ? a.cache.kv_heads : 0) + kvh) * kDim
                                 : a.q + (int64_t)(t_first + idx / R) * a.stride + (int64_t)(kvh * R + idx % R) * kDim;
    const uint4 rx = fetch8<true>(src, m8), ry = fetch8<true>(src, m8 + 8);
    Half x = unpack8<BF16>(rx), y = unpack8<BF16>(ry);
    if (DECODE) {
      const uint16_t* weight = warp < 2 ? a.qw : a.kw;
      const uint4 wx = fetch8<true>(weight, m8), wy = fetch8<true>(weight, m8 + 8);
      int64_t pos = a.positions[b];
      if (pos < 0 || pos >= a.max_positions) {
        if (tid == 0) report(a.status, NQB200_ERR_BAD_INDEX);
        pos = 0;
      }
      norm_turn<BF16>(x, y, wx, wy, angles_of(a.cos_sin + pos * kDim), a.eps, !is_v);
    }
    if (warp < 2) {
      uint4 lo, hi, lo_rest, hi_rest;
      const float f = operand(x, y, lo, hi, lo_rest, hi_rest);
      reinterpret_cast<uint4*>(fx.q[unit])[m8] = lo;
      reinterpret_cast<uint4*>(fx.q[unit])[m8 + 8] = hi;
      if (kRest) {
        reinterpret_cast<uint4*>(fx.rest[unit])[m8] = lo_rest;
        reinterpret_cast<uint4*>(fx.rest[unit])[m8 + 8] = hi_rest;
      }
      if (m8 == 0) fx.unit[unit] = f;
    } else {
      uint2 words, params;
      quantise<BF16>(x, y, words, params);
      if (unit < 10) {
        reinterpret_cast<uint2*>(fx.own[is_v])[m8] = words;
        if (m8 == 0) fx.own_params[is_v] = params;
        const int64_t at = a.rows[b];
        if (group == 0 && at >= 0) {
          const int64_t page = at / a.cache.block;
          if (page < a.cache.pages) {
            const int r = (int)(at - page * a.cache.block);
            uint8_t* base = (is_v ? a.cache.v : a.cache.k) + page_at(a.cache, page, kvh);
            reinterpret_cast<uint2*>(base + r * kData)[m8] = words;
            if (m8 == 0) *reinterpret_cast<uint2*>(base + (int64_t)a.cache.block * kData + r * kParams) = params;
          } else if (m8 == 0) {
            report(a.status, NQB200_ERR_BAD_INDEX);
          }
        }
      }
    }
  }
  __syncthreads();

  const int g = lane >> 2, t4 = lane & 3;
  // word j of a lane's 16 bytes of a key: dimensions 64 (j & 1) + 16 t4 + 8 (j >> 1) .. + 7
  uint32_t qf[4][4];
  // of columns 2 t4 + u: the unit of scores in log2 units, the sums of the query's halves in it, and minus 1024 times the operand's sums
  float f[2], qs[2][2], start[2][2];
  {
    float even[2] = {0.f, 0.f}, odd[2] = {0.f, 0.f};       // of column g, over the lane's dimensions
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 v = *reinterpret_cast<const uint4*>(&fx.q[g][64 * (j & 1) + 16 * t4 + 8 * (j >> 1)]);
      qf[j][0] = v.x; qf[j][1] = v.y; qf[j][2] = v.z; qf[j][3] = v.w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&qf[j][i]));
        (i & 1 ? odd : even)[j & 1] += p.x + p.y;
      }
      if (kRest) {
        const uint4 left = *reinterpret_cast<const uint4*>(&fx.rest[g][64 * (j & 1) + 16 * t4 + 8 * (j >> 1)]);
        const uint32_t lw[4] = {left.x, left.y, left.z, left.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&lw[i]));
          (i & 1 ? odd : even)[j & 1] += p.x + p.y;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) f[u] = a.scale * kLog2e * fx.unit[2 * t4 + u];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        even[h] += __shfl_xor_sync(0xFFFFFFFFu, even[h], o);
        odd[h] += __shfl_xor_sync(0xFFFFFFFFu, odd[h], o);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float p = __shfl_sync(0xFFFFFFFFu, even[h], (2 * t4 + u) * 4), q = __shfl_sync(0xFFFFFFFFu, odd[h], (2 * t4 + u) * 4);
        qs[h][u] = f[u] * fmaf(16.f, q, p);
        start[h][u] = -1024.f * (p + q);
      }
    }
  }
  uint32_t magic;                                  // (out of the compiler's sight, see lift)
  asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));
  // how many keys this lane's columns see, and the fewest of any column
  int sees[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) sees[u] = DECODE ? keys : min(keys, first_pos + token_of(min(2 * t4 + u, cols - 1)) + 1);
  const int all_see = DECODE ? keys : min(keys, first_pos + token_of(0) + 1);

  float ref[2] = {0.f, 0.f}, l[2] = {0.f, 0.f}, L[2][2] = {{0.f, 0.f}, {0.f, 0.f}};     // L[half][column]: sums of weight times level 8
  float O[8][4];                                   // O[4 half + i]: dimensions 64 half + 8 g + 2 i and + 1
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) O[i][e] = 0.f;
  float inv[2] = {power_of_two(126), power_of_two(126)};       // the reciprocals of the columns' units of weight times scale, powers of two

  // row i of a product's 16 keys is key i ^ bit 1 of i
  const int key_g = g ^ ((g >> 1) & 1), kv0 = (2 * t4) ^ (t4 & 1), kv1 = (2 * t4 + 1) ^ (t4 & 1);
  const int koff = key_g * kData + ((t4 ^ ((g >> 1) & 2)) << 4);
  const int voff = kOffV + (((g >> 1) ^ (t4 & 2)) << 4) + (g & 1) * 8;

  bool first = true;
  const auto tile = [&](auto edge, const uint8_t* st, int p0) {
    constexpr bool EDGE = decltype(edge)::value;
    float x[2][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {                  // 16 keys
      const uint4 ka = *reinterpret_cast<const uint4*>(st + u * 16 * kData + koff), kb = *reinterpret_cast<const uint4*>(st + (u * 16 + 8) * kData + koff);
      const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
      float c[2][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Lifted la = lift(wa[j], magic), lb = lift(wb[j], magic);
        if (CTAS == 4) {                           // (again from shared memory rather than in 16 registers)
          const uint4 v = *reinterpret_cast<const uint4*>(&fx.q[g][64 * (j & 1) + 16 * t4 + 8 * (j >> 1)]);
          qf[j][0] = v.x; qf[j][1] = v.y; qf[j][2] = v.z; qf[j][3] = v.w;
        }
        if (j < 2) mma_from(c[j], start[j], la.v[0], lb.v[0], la.v[1], lb.v[1], qf[j][0], qf[j][1]);
        else mma(c[j & 1], la.v[0], lb.v[0], la.v[1], lb.v[1], qf[j][0], qf[j][1]);
        mma(c[j & 1], la.v[2], lb.v[2], la.v[3], lb.v[3], qf[j][2], qf[j][3]);
        if (kRest) {
          const uint4 left = *reinterpret_cast<const uint4*>(&fx.rest[g][64 * (j & 1) + 16 * t4 + 8 * (j >> 1)]);
          mma(c[j & 1], la.v[0], lb.v[0], la.v[1], lb.v[1], left.x, left.y);
          mma(c[j & 1], la.v[2], lb.v[2], la.v[3], lb.v[3], left.z, left.w);
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint2 p = *reinterpret_cast<const uint2*>(st + kOffKP + (u * 16 + 8 * r + key_g) * kParams);
        const float s0 = scale_of<BF16>(p.x), s1 = scale_of<BF16>(p.y), m0 = offset_of<BF16>(p.x), m1 = offset_of<BF16>(p.y);
#pragma unroll
        for (int h = 0; h < 2; ++h)
          x[u][2 * r + h] = fmaf(fmaf(s0, c[0][2 * r + h], s1 * c[1][2 * r + h]), f[h], fmaf(m0, qs[0][h], fmaf(m1, qs[1][h], -ref[h])));
      }
    }
    const auto seen = [&](int u, int e) { return !EDGE || p0 + u * 16 + 8 * (e >> 1) + key_g < sees[e & 1]; };
    if (EDGE) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[u][e] = seen(u, e) ? x[u][e] : -INFINITY;
    }
    uint2 vp[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 2; ++r) vp[u][r] = *reinterpret_cast<const uint2*>(st + kOffVP + (u * 16 + 8 * r + key_g) * kParams);
    float top[2] = {max3(fmaxf(x[0][0], x[0][2]), x[1][0], x[1][2]), max3(fmaxf(x[0][1], x[0][3]), x[1][1], x[1][3])};
    float s_top = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 2; ++r) s_top = max3(s_top, scale_of<BF16>(vp[u][r].x), scale_of<BF16>(vp[u][r].y));      // (a NaN is passed over)
    // The first tile sets the reference.  (What a column sees is a beginning of the keys: one that sees nothing of the first tile sees nothing at all.)
    if (first || __any_sync(0xFFFFFFFFu, top[0] > kLag || top[1] > kLag || s_top * fmaxf(inv[0], inv[1]) > kAhead)) {
      float most[2] = {-INFINITY, -INFINITY};      // log2 of the tile's largest weight times scale, up to one above it
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float s = fmaxf(fmaxf(scale_of<BF16>(vp[u][r].x), scale_of<BF16>(vp[u][r].y)), 0.f), order = (float)((int)(__float_as_uint(s) >> 23) - 126);
#pragma unroll
          for (int h = 0; h < 2; ++h) most[h] = fmaxf(most[h], x[u][2 * r + h] + order);
        }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], o));
          most[h] = fmaxf(most[h], __shfl_xor_sync(0xFFFFFFFFu, most[h], o));
        }
      }
      float far[2];                                // what the sums so far are multiplied by
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float by = first ? (top[h] == -INFINITY ? 0.f : top[h]) : fmaxf(top[h], 0.f), f = first ? 0.f : exp2_fast(-by);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          x[u][h] -= by;
          x[u][2 + h] -= by;
        }
        ref[h] += by;
        l[h] *= f;
        L[0][h] *= f;
        L[1][h] *= f;
        // the unit: from 2^-110 to 2^125, no less than what the sums so far ask for
        const int before = 127 - (int)(__float_as_uint(inv[h]) >> 23);
        const int order = (int)ceilf(fminf(fmaxf((first ? most[h] : fmaxf(most[h], (float)before)) - by, -110.f), 125.f));
        inv[h] = power_of_two(-order);
        far[h] = first ? 0.f : exp2_fast((float)(before - order) - by);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) O[i][e] *= far[e & 1];
    }
    uint32_t w[2][2][2];                           // [16 keys][half][rows of 8]: weights as the second operand
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float p[2], q[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) { p[h] = exp2_fast(x[u][2 * r + h]); q[h] = p[h] * inv[h]; l[h] += p[h]; }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t par = half ? vp[u][r].y : vp[u][r].x;
          const float s = scale_of<BF16>(par), o = fmaf(8.f, s, offset_of<BF16>(par));
          // a key that a column does not see has no part in it, even where its value is not a number
          if (EDGE) {
#pragma unroll
            for (int h = 0; h < 2; ++h) L[half][h] = seen(u, 2 * r + h) ? fmaf(p[h], o, L[half][h]) : L[half][h];
            w[u][half][r] = transpose8(pack2(seen(u, 2 * r) ? q[0] * s : 0.f, seen(u, 2 * r + 1) ? q[1] * s : 0.f));
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) L[half][h] = fmaf(p[h], o, L[half][h]);
            w[u][half][r] = transpose8(pack2(q[0] * s, q[1] * s));
          }
        }
      }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint8_t* vs = st + u * 16 * kData + voff;
      const uint2 va = *reinterpret_cast<const uint2*>(vs + kv0 * kData), vb = *reinterpret_cast<const uint2*>(vs + kv1 * kData);
      const uint2 vc = *reinterpret_cast<const uint2*>(vs + (kv0 + 8) * kData), vd = *reinterpret_cast<const uint2*>(vs + (kv1 + 8) * kData);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t a_ = half ? va.y : va.x, b_ = half ? vb.y : vb.x, c_ = half ? vc.y : vc.x, d_ = half ? vd.y : vd.x;
        // dimensions of the word's low and high 16 bits, of two keys each
        const Lifted lo0 = levels(__byte_perm(a_, b_, 0x5410), magic), hi0 = levels(__byte_perm(a_, b_, 0x7632), magic);
        const Lifted lo1 = levels(__byte_perm(c_, d_, 0x5410), magic), hi1 = levels(__byte_perm(c_, d_, 0x7632), magic);
        const uint32_t b0 = w[u][half][0], b1 = w[u][half][1];
#pragma unroll
        for (int i = 0; i < 4; ++i) mma(O[4 * half + i], lo0.v[i], hi0.v[i], lo1.v[i], hi1.v[i], b0, b1);
      }
    }
  };

  int stage = 0;
  for (int t = t0 + warp; t < t1; t += kWarps) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();                                  // the tile is there for every lane, the one before it is no longer read
    load(t + (STAGES - 1) * kWarps, stage == 0 ? STAGES - 1 : stage - 1);
    uint8_t* st = ring + stage * kStage;
    const int p0 = t * kTile;
    if (DECODE && t == tiles - 1) {                // the step's own key and value go into the tile
      const int r = keys - 1 - p0, c = lane & 15, which = lane >> 4;
      reinterpret_cast<uint32_t*>(st + (which ? kOffV : 0) + r * kData + (((c >> 2) ^ ((r >> 1) & 2)) << 4))[c & 3] = fx.own[which][c];
      if (c == 0) *reinterpret_cast<uint2*>(st + (which ? kOffVP : kOffKP) + r * kParams) = fx.own_params[which];
      __syncwarp();
    }
    if (p0 + kTile > all_see) tile(std::true_type(), st, p0); else tile(std::false_type(), st, p0);
    first = false;
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();

  // the warps' shares over their rings
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], o);
      L[0][h] += __shfl_xor_sync(0xFFFFFFFFu, L[0][h], o);
      L[1][h] += __shfl_xor_sync(0xFFFFFFFFu, L[1][h], o);
    }
  }
  const float unit_v[2] = {1.f / inv[0], 1.f / inv[1]};
  float* po = reinterpret_cast<float*>(ring);      // [column][kOS]
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int half = i >> 2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float2 v = make_float2(fmaf(O[i][h], unit_v[h], L[half][h]), fmaf(O[i][2 + h], unit_v[h], L[half][h]));
      *reinterpret_cast<float2*>(po + (2 * t4 + h) * kOS + 64 * half + 8 * g + 2 * (i & 3)) = v;
    }
  }
  if (lane < 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) { fx.m[warp][2 * lane + h] = l[h] == 0.f ? -INFINITY : ref[h]; fx.l[warp][2 * lane + h] = l[h]; }
  }
  __syncthreads();
  const auto finish = [&](int c, int d, float o, float sum, float top) {
    const int idx = group * kCols + c;
    const int64_t row = (int64_t)(t_first + idx / R) * a.heads + kvh * R + idx % R;
    if (a.parts > 1) {
      float* share = a.shares + (row * a.parts + blockIdx.x / csize) * kShare;
      share[d] = o;
      if (d == 0) { share[kDim] = top; share[kDim + 1] = sum; }
    } else {
      a.out[row * kDim + d] = float_to_raw16<BF16>(sum == 0.f ? 0.f : o / sum);
    }
  };
  for (int c = 0; c < cols; ++c) {
    float top = -INFINITY, o = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, fx.m[w][c]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = fx.m[w][c] == top ? 1.f : exp2_fast(fx.m[w][c] - top);      // 0: a warp without keys
      o += f * reinterpret_cast<const float*>(smem + w * (STAGES * kStage))[c * kOS + tid];
      sum += f * fx.l[w][c];
    }
    if (csize == 1) {
      finish(c, tid, o, sum, top);
    } else {
      fx.out[c][tid] = o;
      if (tid == 0) { fx.cm[c] = top; fx.cl[c] = sum; }
    }
  }
  if (csize == 1) return;
  cl.sync();
  for (int e = rank * kThreads + tid; e < cols * kDim; e += csize * kThreads) {
    const int c = e / kDim, d = e % kDim;
    float pm[8], pl[8], po8[8], top = -INFINITY, o = 0.f, sum = 0.f;              // all of the cluster's shares at once
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const Fixed* s = cl.map_shared_rank(&fx, k < csize ? k : 0);
      pm[k] = k < csize ? s->cm[c] : -INFINITY;
      pl[k] = s->cl[c];
      po8[k] = s->out[c][d];
      top = fmaxf(top, pm[k]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = k >= csize ? 0.f : pm[k] == top ? 1.f : exp2_fast(pm[k] - top);
      o += f * po8[k];
      sum += f * pl[k];
    }
    finish(c, d, o, sum, top);
  }
  cl.sync();                                       // peers may still read this CTA's shared memory
}

// The shares of a row, a CTA per (token, query head), in their order.  A lane has the maximum and the sum of two of up to 64 shares.
template <bool BF16>
__global__ void __launch_bounds__(kDim) kv4_shares_kernel(const float* __restrict__ shares, uint16_t* __restrict__ out, int parts) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int64_t row = blockIdx.x;
  const float* s = shares + row * parts * kShare;
  const int lane = threadIdx.x & 31;
  float m[2], f[2], sum = 0.f, top = -INFINITY, o = 0.f, v[8];       // v: the first shares' sums, under way beside the maxima
#pragma unroll
  for (int p = 0; p < 8; ++p) v[p] = p < parts ? s[p * kShare + threadIdx.x] : 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int p = lane + 32 * k;
    m[k] = p < parts ? s[p * kShare + kDim] : -INFINITY;
    f[k] = p < parts ? s[p * kShare + kDim + 1] : 0.f;
    top = fmaxf(top, m[k]);
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float by = m[k] == top ? 1.f : exp2f(m[k] - top);
    sum += by * f[k];
    f[k] = by;
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const float by = __shfl_sync(0xFFFFFFFFu, f[0], p);
    if (p < parts) o += by * v[p];
  }
#pragma unroll 8
  for (int p = 8; p < parts; ++p) o += __shfl_sync(0xFFFFFFFFu, p < 32 ? f[0] : f[1], p & 31) * s[p * kShare + threadIdx.x];
  out[row * kDim + threadIdx.x] = float_to_raw16<BF16>(sum == 0.f ? 0.f : o / sum);
}

}  // namespace

int kv4::add_shares(const float* shares, uint16_t* out, int64_t rows, int parts, bool bf16, cudaStream_t st) {
  return launch_overlapped(bf16 ? kv4_shares_kernel<true> : kv4_shares_kernel<false>, dim3((unsigned)rows), dim3(kDim), 0, st, shares, out, parts);
}

namespace {

// How a call is split: CTAs of a cluster, CTAs that share an SM, clusters of a sequence.  Clusters of 1, 2, 4, 8 CTAs that are resident with 2, 3
// and 4 CTAs to an SM:
constexpr int kResident[4][3] = {{296, 444, 592}, {148, 222, 296}, {71, 104, 142}, {33, 48, 66}};
constexpr int kMostParts = 16;
struct Split { int csize, ctas, parts; };
// `keys`: the most that a sequence may see; a unit: eight columns of a key/value head of a sequence.
// The fewer CTAs share an SM, the more registers each has: a CTA per 128 keys (a tile per warp) as long as the clusters are resident three to an SM,
// and two to an SM where they still are.  Units of 1500 keys, us, with 2, 3, 4 to an SM: 192 (clusters of two) 28.5, 18.8, 21.8; 256 (of 2000) 25.1,
// 31.1, 37.3; 360 37.1, 26.6, 33.0.  Four to an SM is for what then takes one turn instead of two: 512 of 4000 80, 87, 75, and where turns
// are many; 880 units 55.7, 48.9, 54.1; 2048 of 800 87, 72.7, 70.9.
// Where clusters of eight leave half of the chip idle, a sequence goes over several of them, down to 128 keys a CTA, and a second kernel adds their
// shares (3 us).  8 key/value heads, over one cluster, two and four: 2048 keys 7.8, 9.6, 9.0; 4000 9.7, 10.4, 9.2; 8000 12.3, 12.3, 10.3;
// 32000 34, 27, 18.7.
Split split(int64_t units, int64_t keys) {
  Split s = {1, 4, 1};
  int row = 0;
  while (row < 3 && units <= kResident[row + 1][1] && keys > (int64_t)s.csize * kWarps * kTile) { s.csize *= 2; ++row; }
  if (row == 3 && keys >= 4096)
    while (s.parts < kMostParts && units * s.parts * 2 <= kResident[3][0] && keys >= 8 * s.parts * 2 * 128) s.parts *= 2;
  const auto turns = [&](int ctas) { return (units * s.parts + kResident[row][ctas - 2] - 1) / kResident[row][ctas - 2]; };
  if (turns(2) == 1) s.ctas = 2;
  else if (turns(3) * 4 < turns(4) * 5) s.ctas = 3;
  return s;
}

int groups_of(int64_t tokens, int64_t heads, int64_t kv_heads) { return (int)((tokens * (heads / kv_heads) + kCols - 1) / kCols); }

// Units that have columns: sequences shorter than the longest have fewer, and half a unit each is lost at their ends.
int64_t units_of(int64_t batch, int64_t tokens, int64_t groups, int64_t heads, int64_t kv_heads) {
  const int64_t full = batch * groups, some = tokens * (heads / kv_heads) / kCols + (batch + 1) / 2;
  return kv_heads * (tokens > batch && some < full ? some : full);
}

template <bool BF16, bool DECODE, int CTAS> int launch_ctas(const Args& a, int csize, int64_t batch, cudaStream_t st) {
  constexpr auto kernel = kv4_rows_kernel<BF16, DECODE, CTAS>;
  constexpr int smem = smem_bytes(stages_of(CTAS));
  if (!allow_smem<kernel>(smem)) return NQB200_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(csize * a.parts), (unsigned)(a.cache.kv_heads * a.groups), (unsigned)batch);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)csize;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) { cudaGetLastError(); return NQB200_ERR_LAUNCH; }
  return NQB200_OK;
}
template <bool BF16, bool DECODE> int launch_t(Args& a, int64_t batch, int64_t tokens, int64_t keys, cudaStream_t st) {
  const Split s = split(units_of(batch, tokens, a.groups, a.heads, a.cache.kv_heads), keys);
  a.parts = s.parts;
  a.shift = (a.cache.block & (a.cache.block - 1)) == 0 ? __builtin_ctz((unsigned)a.cache.block) : -1;
  const int rc = s.ctas == 2   ? launch_ctas<BF16, DECODE, 2>(a, s.csize, batch, st)
                 : s.ctas == 3 ? launch_ctas<BF16, DECODE, 3>(a, s.csize, batch, st)
                               : launch_ctas<BF16, DECODE, 4>(a, s.csize, batch, st);
  if (rc != NQB200_OK || s.parts == 1) return rc;
  return add_shares(a.shares, a.out, tokens * a.heads, s.parts, BF16, st);
}
template <bool DECODE> int launch(Args& a, int64_t batch, int64_t tokens, int64_t keys, int dtype, cudaStream_t st) {
  return dtype == NQB200_BF16 ? launch_t<true, DECODE>(a, batch, tokens, keys, st) : launch_t<false, DECODE>(a, batch, tokens, keys, st);
}
size_t scratch_bytes_of(int64_t batch, int64_t tokens, int64_t max_len, int64_t keys, int64_t heads, int64_t kv_heads) {
  const Split s = split(units_of(batch, tokens, groups_of(max_len, heads, kv_heads), heads, kv_heads), keys);
  return s.parts > 1 ? (size_t)(tokens * heads * s.parts * kShare) * sizeof(float) : 0;
}
bool heads_fit(int64_t heads, int64_t kv_heads) { return kv_heads > 0 && kv_heads <= 4096 && heads > 0 && heads <= 65535 && heads % kv_heads == 0; }
// (keys are numbered in 32 bits, up to the end of the last tile)
bool table_fits(int64_t width, int64_t block) { return width > 0 && block > 0 && width <= (INT32_MAX - 256) / block; }

}  // namespace
}  // namespace nqb200

using namespace nqb200;

static int check_heads(const nqb200_kv4* cache, int64_t heads, int64_t width, int dtype) {
  const int rc = kv4::check_cache(cache);
  if (rc != NQB200_OK) return rc;
  if (!heads_fit(heads, cache->kv_heads) || !table_fits(width, cache->block_size)) return NQB200_ERR_BAD_SHAPE;
  return dtype == NQB200_F16 || dtype == NQB200_BF16 ? NQB200_OK : NQB200_ERR_BAD_DTYPE;
}

extern "C" size_t nqb200_kv4_decode_scratch_bytes(int64_t table_width, int64_t block_size, int64_t batch, int64_t num_q_heads, int64_t kv_heads) {
  if (!heads_fit(num_q_heads, kv_heads) || !table_fits(table_width, block_size) || batch <= 0 || batch > 65535) return 0;
  return scratch_bytes_of(batch, batch, 1, table_width * block_size, num_q_heads, kv_heads);
}

extern "C" int nqb200_kv4_decode_attention(const void* qkv, int64_t row_stride, const void* q_weight, const void* k_weight, const float* cos_sin,
                                           int64_t max_positions, const int64_t* positions, const int64_t* rows, const nqb200_kv4* cache,
                                           const int32_t* table, int64_t table_width, const int32_t* ctx, void* out, int64_t batch, int64_t num_q_heads,
                                           float scale, float eps, int dtype, void* scratch, size_t scratch_bytes, int* status, void* stream) {
  const int rc = check_heads(cache, num_q_heads, table_width, dtype);
  if (rc != NQB200_OK) return rc;
  const int groups = groups_of(1, num_q_heads, cache->kv_heads);
  if (batch < 0 || batch > 65535 || cache->kv_heads * groups > 65535 || max_positions <= 0 || row_stride < (num_q_heads + 2 * cache->kv_heads) * kv4::kDim || row_stride % 8 != 0)
    return NQB200_ERR_BAD_SHAPE;
  if (batch == 0) return NQB200_OK;
  if (!qkv || !q_weight || !k_weight || !cos_sin || !positions || !rows || !table || !ctx || !out) return NQB200_ERR_NULL_POINTER;
  if (!aligned16(qkv) || !aligned16(q_weight) || !aligned16(k_weight) || !aligned16(cos_sin) || !aligned16(out)) return NQB200_ERR_MISALIGNED;
  const size_t need = nqb200_kv4_decode_scratch_bytes(table_width, cache->block_size, batch, num_q_heads, cache->kv_heads);
  if (need > 0 && (!scratch || scratch_bytes < need)) return NQB200_ERR_WORKSPACE;
  if (need > 0 && !aligned16(scratch)) return NQB200_ERR_MISALIGNED;
  Args a = {};
  a.q = (const uint16_t*)qkv; a.stride = row_stride; a.qw = (const uint16_t*)q_weight; a.kw = (const uint16_t*)k_weight;
  a.cos_sin = cos_sin; a.max_positions = max_positions; a.positions = positions; a.rows = rows; a.cache = kv4::cache_of(cache);
  a.table = table; a.width = (int)table_width; a.ctx = ctx; a.out = (uint16_t*)out; a.heads = (int)num_q_heads; a.groups = groups; a.max_len = 1;
  a.scale = scale; a.eps = eps; a.status = status; a.shares = (float*)scratch;
  return launch<true>(a, batch, batch, table_width * cache->block_size, dtype, (cudaStream_t)stream);
}

// Few rows or many; what does not fit into the grid of the way for few goes the other way.
static bool prompt_goes_umma(int64_t batch, int64_t T, int64_t max_len, int64_t max_ctx, int64_t tiles, int64_t heads, int64_t kv_heads) {
  return kv_heads * groups_of(max_len, heads, kv_heads) > 65535 || kv4::prompt_umma_faster(batch, T, max_len, max_ctx, tiles, heads, kv_heads);
}

extern "C" size_t nqb200_kv4_prompt_scratch_bytes(int64_t batch, int64_t T, int64_t max_len, int64_t max_ctx, int64_t tiles, int64_t num_q_heads, int64_t kv_heads) {
  if (!heads_fit(num_q_heads, kv_heads) || batch <= 0 || batch > 65535 || T <= 0 || max_len <= 0 || max_len > T || max_ctx < max_len || max_ctx > INT32_MAX - 256 || tiles <= 0 ||
      tiles > kv4::kMostTiles)
    return 0;
  if (prompt_goes_umma(batch, T, max_len, max_ctx, tiles, num_q_heads, kv_heads))
    return kv4::prompt_umma_scratch_bytes(batch, T, max_len, max_ctx, tiles, num_q_heads, kv_heads);
  return scratch_bytes_of(batch, T, max_len, max_ctx, num_q_heads, kv_heads);
}

extern "C" const char* nqb200_kv4_prompt_kernel_name(int64_t batch, int64_t T, int64_t max_len, int64_t max_ctx, int64_t tiles, int64_t num_q_heads, int64_t kv_heads) {
  if (!heads_fit(num_q_heads, kv_heads) || batch <= 0 || T <= 0 || max_len <= 0 || max_ctx < max_len || tiles <= 0) return "invalid";
  return prompt_goes_umma(batch, T, max_len, max_ctx, tiles, num_q_heads, kv_heads) ? "tiles_tcgen05" : "rows";
}

extern "C" int nqb200_kv4_prompt_attention(const void* q, int64_t q_stride, const nqb200_kv4* cache, const int32_t* table, int64_t table_width,
                                           const int32_t* cu, const int32_t* pos0, void* out, int64_t batch, int64_t T, int64_t max_len, int64_t max_ctx,
                                           int64_t tiles, int64_t num_q_heads, float scale, int dtype, void* scratch, size_t scratch_bytes, int* status, void* stream) {
  const int rc = check_heads(cache, num_q_heads, table_width, dtype);
  if (rc != NQB200_OK) return rc;
  if (batch < 0 || batch > 65535 || T < 0 || T > INT32_MAX / num_q_heads || max_len < 0 || (T > 0 && max_len > T) || max_ctx < max_len || max_ctx > INT32_MAX - 256 || tiles < 0 || tiles > kv4::kMostTiles ||
      q_stride < num_q_heads * kv4::kDim || q_stride % 8 != 0)
    return NQB200_ERR_BAD_SHAPE;
  if (batch == 0 || T == 0) return NQB200_OK;
  const int64_t groups = groups_of(max_len, num_q_heads, cache->kv_heads);
  if (max_len == 0 || tiles == 0) return NQB200_ERR_BAD_SHAPE;
  const bool umma = prompt_goes_umma(batch, T, max_len, max_ctx, tiles, num_q_heads, cache->kv_heads);
  if (!q || !table || !cu || !pos0 || !out) return NQB200_ERR_NULL_POINTER;
  if (!aligned16(q) || !aligned16(out)) return NQB200_ERR_MISALIGNED;
  const size_t need = nqb200_kv4_prompt_scratch_bytes(batch, T, max_len, max_ctx, tiles, num_q_heads, cache->kv_heads);
  if (need > 0 && (!scratch || scratch_bytes < need)) return NQB200_ERR_WORKSPACE;
  if (need > 0 && !aligned16(scratch)) return NQB200_ERR_MISALIGNED;
  if (umma)
    return kv4::prompt_umma((const uint16_t*)q, q_stride, cache, table, table_width, cu, pos0, (uint16_t*)out, batch, T, max_len, max_ctx, tiles, num_q_heads, scale, dtype,
                            scratch, status, (cudaStream_t)stream);
  Args a = {};
  a.q = (const uint16_t*)q; a.stride = q_stride; a.cache = kv4::cache_of(cache); a.table = table; a.width = (int)table_width; a.cu = cu; a.pos0 = pos0;
  a.out = (uint16_t*)out; a.heads = (int)num_q_heads; a.groups = (int)groups; a.tokens = (int)T; a.max_len = (int)max_len; a.max_ctx = (int)max_ctx; a.scale = scale; a.status = status; a.shares = (float*)scratch;
  return launch<false>(a, batch, T, max_ctx, dtype, (cudaStream_t)stream);
}
