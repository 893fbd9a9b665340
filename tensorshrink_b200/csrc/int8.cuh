// 8-bit integers with a scale per row, shared by the quantiser and the product.
#pragma once

#include "fp4.cuh"

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

using fp4::Elem;

// Columns 8 c .. 8 c + 7 of a row as words (four, or eight of fp32); zeros behind the last one.
template <int DT, bool AL>
__device__ __forceinline__ void load8(const typename Elem<DT>::T* row, int c, int64_t cols, uint32_t (&w)[DT == TS_F32 ? 8 : 4]) {
  constexpr int N = DT == TS_F32 ? 8 : 4;
  const int64_t left = cols - 8 * (int64_t)c;
  const auto* p = row + 8 * (int64_t)c;
  if (left >= 8) {
    if constexpr (AL) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + i);
        w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
      }
    } else if constexpr (DT == TS_F32) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = __ldg(p + i);
    } else {
      // the words that hold the eight elements: a fifth one where they start in the middle of one
      const uintptr_t at = reinterpret_cast<uintptr_t>(p);
      const uint32_t* q = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
      uint32_t u[5];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = __ldg(q + i);
      u[4] = at & 2 ? __ldg(q + 4) : 0;
      const unsigned by = at & 2 ? 16 : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(u[i], u[i + 1], by);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) {
      if (DT == TS_F32) w[i % N] = (uint32_t)p[i];
      else w[(i / 2) % N] |= (uint32_t)p[i] << (16 * (i & 1));
    }
}

// Largest magnitude of a chunk, as fp32 bits (of a NaN or an infinity: at least 0x7F800000).
template <int DT, int N>
__device__ __forceinline__ uint32_t top8(const uint32_t (&w)[N]) {
  uint32_t m = 0;
  if constexpr (DT == TS_F32) {
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
    return m;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
    m = max(m & 0xFFFFu, m >> 16);
    // (fp16: infinities and NaN keep their kind in fp32)
    return __float_as_uint(Elem<DT>::f((uint16_t)m));
  }
}

// Eight codes x r to nearest even: what adding 1.5 * 2^23 leaves in the sums' low bits.
template <int DT, int N>
__device__ __forceinline__ uint2 codes8(const uint32_t (&w)[N], float r) {
  const Two rr = two(r, r), magic = two(12582912.f, 12582912.f);
  float2 q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    Two f;
    if constexpr (DT == TS_F32) f = two(__uint_as_float(w[(2 * i) % N]), __uint_as_float(w[(2 * i + 1) % N]));
    else f = two(Elem<DT>::f((uint16_t)(w[i] & 0xFFFFu)), Elem<DT>::f((uint16_t)(w[i] >> 16)));
    q[i] = both(add2(mul2_rn(f, rr), magic));
  }
  auto pack = [](float2 a, float2 b) {
    return prmt(prmt(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), prmt(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040),
                0x5410);
  };
  return make_uint2(pack(q[0], q[1]), pack(q[2], q[3]));
}

int check_tensor(const ts_int8_tensor* t, const char* what);

}  // namespace int8
}  // namespace ts
