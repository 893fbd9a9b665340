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

// Element types of what is quantised.
template <int DT>
struct Elem;
template <>
struct Elem<TS_F16> {
  using T = uint16_t;
  static constexpr uint32_t kInf = 0x7C00u;
  static __device__ float f(uint16_t v) { return __half2float(__ushort_as_half(v)); }
};
template <>
struct Elem<TS_BF16> {
  using T = uint16_t;
  static constexpr uint32_t kInf = 0x7F80u;
  static __device__ float f(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
};
template <>
struct Elem<TS_F32> {
  using T = uint32_t;
  static constexpr uint32_t kInf = 0x7F800000u;
  static __device__ float f(uint32_t v) { return __uint_as_float(v); }
};

// A lane's 16 elements as words (8, or 16 of fp32); of rows that start in the
// middle of a word, also the first element of row `lane` (lanes 0 to 3).
template <int DT>
struct Lane {
  static constexpr int N = DT == TS_F32 ? 16 : 8;
  uint32_t w[N];
  uint32_t e;
};

// Largest magnitude as the type's bits (a NaN or infinity: at least kInf).
template <int DT>
__device__ __forceinline__ uint32_t top_bits(const Lane<DT>& v) {
  uint32_t m = 0;
  if constexpr (DT == TS_F32) {
#pragma unroll
    for (int i = 0; i < Lane<DT>::N; ++i) m = max(m, v.w[i] & 0x7FFFFFFFu);
    return m;
  } else {
#pragma unroll
    for (int i = 0; i < Lane<DT>::N; ++i) m = __vmaxu2(m, v.w[i] & 0x7FFF7FFFu);
    return max(m & 0xFFFFu, m >> 16);
  }
}

// Element i of a lane in fp32.
template <int DT>
__device__ __forceinline__ float elem(const Lane<DT>& v, int i) {
  if (DT == TS_F32) return __uint_as_float(v.w[i % Lane<DT>::N]);
  const uint32_t w = v.w[(i / 2) % Lane<DT>::N];
  if (DT == TS_BF16) return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return i & 1 ? f.y : f.x;
}

// Codes (`out`) and scale (returned) of a lane's 16 columns: a block of nvfp4,
// whose tensor scale is g and to_scale = 1 / (6 g); half a block of mxfp4, the
// neighbouring lane having the other. A whole warp calls it.
template <int DT, bool NV>
__device__ __forceinline__ uint32_t quantise16(const Lane<DT>& v, float g, float to_scale, uint2& out) {
  using E = Elem<DT>;
  uint32_t top = top_bits<DT>(v);
  if (!NV) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  out = make_uint2(0, 0);
  if (top >= E::kInf) return NV ? 0x7Fu : 0xFFu;
  const float amax = E::f((typename E::T)top);
  float r;
  uint32_t sc;
  if (NV) {
    sc = __nv_cvt_float_to_fp8(fminf(__fmul_rn(amax, to_scale), 448.f), __NV_SATFINITE, __NV_E4M3);
    const float sf = e4m3_value((uint8_t)sc);
    r = sf > 0.f ? __frcp_rn(__fmul_rn(sf, g)) : 0.f;
  } else {
    const int e = (int)(__float_as_uint(amax) >> 23) - 2;
    sc = (uint32_t)max(e, 0);
    r = __uint_as_float((254u - sc) << 23);
  }
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = elem<DT>(v, i);
  out.x = to_e2m1x8(f, r);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = elem<DT>(v, 8 + i);
  out.y = to_e2m1x8(f, r);
  return sc;
}

// Checks a tensor's description (`what` names it in messages).
int check_tensor(const ts_fp4_tensor* t, const char* what);

}  // namespace fp4
}  // namespace ts
