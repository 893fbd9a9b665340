// Microscaled 4-bit floating point: formats, scale layout and conversions
// shared by the quantiser and the product.
#pragma once

#include <cuda_fp8.h>

#include "sm100.cuh"

namespace ts {
namespace fp4 {

constexpr int kColPad = 64;        // columns are padded to a multiple of this
constexpr int kTileRows = 128;     // rows of a scale tile
constexpr int kTileBytes = 512;    // 128 rows x 4 blocks
constexpr float kMinScale = 7.888609052210118e-31f;   // 2^-100
constexpr float kMaxScale = 3.323069989616176e35f;    // 2^118

__host__ __device__ inline int block_of(int format) { return format == TS_NVFP4 ? 16 : 32; }
__host__ __device__ inline int64_t padded_cols(int64_t cols) { return (cols + kColPad - 1) / kColPad * kColPad; }
// Scale tiles along a row.
__host__ __device__ inline int64_t scale_tiles(int64_t cols, int format) {
  return (padded_cols(cols) / block_of(format) + 3) / 4;
}

// Byte of (row, block j) for `kt` scale tiles along a row.
__device__ __forceinline__ int64_t scale_at(int64_t row, int64_t j, int64_t kt) {
  return ((row >> 7) * kt + (j >> 2)) * kTileBytes + (row & 31) * 16 + ((row & 127) >> 5) * 4 + (j & 3);
}

// A usable tensor scale: a NaN or a value outside [2^-100, 2^118] is clamped,
// so that s * g and its reciprocal stay finite normal numbers.
__device__ __forceinline__ float usable_scale(const float* g) {
  return g == nullptr ? 1.f : fminf(fmaxf(*g, kMinScale), kMaxScale);
}

__device__ __forceinline__ float e4m3_value(uint8_t b) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}

__device__ __forceinline__ float e8m0_value(uint8_t b) {
  if (b == 0xFF) return __uint_as_float(0x7FC00000u);
  return b == 0 ? __uint_as_float(0x00400000u) : __uint_as_float((uint32_t)b << 23);
}

// Eight E2M1 codes of x[0..7] * r, nearest even, saturating to +-6.
__device__ __forceinline__ uint32_t to_e2m1x8(const float (&x)[8], float r) {
  uint32_t d;
  asm("{\n .reg .b8 b0, b1, b2, b3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      " mov.b32 %0, {b0, b1, b2, b3};\n}"
      : "=r"(d)
      : "f"(__fmul_rn(x[0], r)), "f"(__fmul_rn(x[1], r)), "f"(__fmul_rn(x[2], r)), "f"(__fmul_rn(x[3], r)),
        "f"(__fmul_rn(x[4], r)), "f"(__fmul_rn(x[5], r)), "f"(__fmul_rn(x[6], r)), "f"(__fmul_rn(x[7], r)));
  return d;
}

// The eight E2M1 values of a word of codes, as four pairs of fp16.
__device__ __forceinline__ void from_e2m1x8(uint32_t d, uint32_t (&h)[4]) {
  asm("{\n .reg .b8 b0, b1, b2, b3;\n mov.b32 {b0, b1, b2, b3}, %4;\n"
      " cvt.rn.f16x2.e2m1x2 %0, b0;\n cvt.rn.f16x2.e2m1x2 %1, b1;\n"
      " cvt.rn.f16x2.e2m1x2 %2, b2;\n cvt.rn.f16x2.e2m1x2 %3, b3;\n}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(d));
}

// Checks a tensor's description (`what` names it in messages).
int check_tensor(const ts_fp4_tensor* t, const char* what);

}  // namespace fp4
}  // namespace ts
