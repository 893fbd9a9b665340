// 8-bit integers with a scale per row, shared by the quantiser and the product.
#pragma once

#include "sm100.cuh"

namespace ts {
namespace int8 {

constexpr int64_t kMaxCols = 131072;   // 127^2 of them sum to less than 2^31
static_assert(127 * 127 * kMaxCols < ((int64_t)1 << 31), "sums of products in 32 bits");

__host__ __device__ inline int64_t padded_cols(int64_t cols) { return (cols + 15) / 16 * 16; }

// Scale of a row (or block) whose largest magnitude is `top`: never so small
// that its reciprocal leaves fp32's normal range.
__device__ __forceinline__ float scale_of(float top) {
  return fmaxf(__fmul_rn(top, (float)(1.0 / 127.0)), 7.888609052210118e-31f);   // 2^-100
}

int check_tensor(const ts_int8_tensor* t, const char* what);

}  // namespace int8
}  // namespace ts
