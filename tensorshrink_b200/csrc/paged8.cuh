// The paged key-value cache held in 8 bits: addressing and codes, shared by its kernels.
#pragma once

#include <cuda_fp8.h>

#include "paged.cuh"

namespace ts {
namespace paged8 {

struct Cache {
  uint8_t* k;
  uint8_t* v;
  int64_t page_stride, head_stride, token_stride;   // bytes, the same for k and v
  float* k_scales;
  float* v_scales;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* seq_lens;
  int batch, n_kv, head_dim, page_size, num_pages, max_pages, block;
  int blocks;          // of a page
};

// Checks the description of a cache and fills the device view.
int make_cache(const ts_paged_cache8* c, Cache* out);

__device__ __forceinline__ int64_t row_at(const Cache& c, int page, int h, int off) {
  return (int64_t)page * c.page_stride + (int64_t)h * c.head_stride + (int64_t)off * c.token_stride;
}
__device__ __forceinline__ int64_t scale_at(const Cache& c, int page, int h, int blk) {
  return ((int64_t)page * c.n_kv + h) * c.blocks + blk;
}

// The largest magnitude of a code, and the scale of values up to `top`: never so
// small that its reciprocal leaves fp32's normal range.
template <bool E4M3>
__device__ __forceinline__ float scale_of(float top) {
  return fmaxf(__fmul_rn(top, E4M3 ? (float)(1.0 / 448.0) : (float)(1.0 / 127.0)), 7.888609052210118e-31f);   // 2^-100
}

// Four codes of values that were divided by their scale, at most the largest code's size
// (give or take fp32's rounding, which stays below half a step): to nearest even. An
// integer is what adding 1.5 * 2^23 leaves in the sum's low bits.
template <bool E4M3>
__device__ __forceinline__ uint32_t encode4(Two a, Two b) {
  if constexpr (E4M3) {
    const float2 x = both(a), y = both(b);
    uint32_t w;
    asm("{\n .reg .b16 lo, hi;\n cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n"
        " mov.b32 %0, {lo, hi};\n}" : "=r"(w) : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
    return w;
  } else {
    const Two magic = two(12582912.f, 12582912.f);
    const float2 x = both(add2(a, magic)), y = both(add2(b, magic));
    return prmt(prmt(__float_as_uint(x.x), __float_as_uint(x.y), 0x0040), prmt(__float_as_uint(y.x), __float_as_uint(y.y), 0x0040),
                0x5410);
  }
}

// The values of four codes, unscaled.
template <bool E4M3>
__device__ __forceinline__ void decode4(uint32_t w, float (&f)[4]) {
  if constexpr (E4M3) {
    uint32_t lo, hi;
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
        : "=r"(lo), "=r"(hi) : "r"(w));
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    f[0] = x.x; f[1] = x.y; f[2] = y.x; f[3] = y.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(w >> (8 * i));
  }
}

struct AppendArgs {
  Cache c;
  const uint16_t* k;
  const uint16_t* v;
  int64_t kb, kt, kh, vb, vt, vh;   // element strides of sequence, token, head
  int64_t tokens;                   // of each sequence, or packed in all
  const int32_t* offsets;
  const int32_t* n_new;
  const int64_t* first;
  const float* cos_t;
  const float* sin_t;
  int64_t rope_rows;
};
// Launches the append of arguments that were checked; `most`: the tokens of a
// sequence at most.
int launch_append(const AppendArgs& a, int dtype, int code, int64_t most, cudaStream_t st);

}  // namespace paged8
}  // namespace ts
