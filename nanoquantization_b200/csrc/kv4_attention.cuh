// What the two ways of attending to the 4-bit cache share: few query rows (kv4_attention.cu) and many (kv4_prompt.cu).
#pragma once
#include "kv4.cuh"

namespace nqb200 {
namespace kv4 {

constexpr int kMostTiles = 1 << 24;   // of 128 keys, in a prompt call: a terabyte of scratch
constexpr int kShare = kDim + 4;      // floats of a row's share of its keys: sums, maximum (log2 units), sum of weights

// out[row] = the sum of the row's shares (64 at most), in their order, over its sum of weights; 0 where there is no key.
int add_shares(const float* shares, uint16_t* out, int64_t rows, int parts, bool bf16, cudaStream_t st);

bool prompt_umma_faster(int64_t batch, int64_t tokens, int64_t max_len, int64_t max_ctx, int64_t tiles, int64_t heads, int64_t kv_heads);
size_t prompt_umma_scratch_bytes(int64_t batch, int64_t tokens, int64_t max_len, int64_t max_ctx, int64_t tiles, int64_t heads, int64_t kv_heads);
int prompt_umma(const uint16_t* q, int64_t q_stride, const nqb200_kv4* cache, const int32_t* table, int64_t width, const int32_t* cu, const int32_t* pos0,
                uint16_t* out, int64_t batch, int64_t tokens, int64_t max_len, int64_t max_ctx, int64_t tiles, int64_t heads, float scale, int dtype, void* scratch,
                int* status, cudaStream_t st);

}  // namespace kv4
}  // namespace nqb200
