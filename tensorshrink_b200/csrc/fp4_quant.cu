// Quantisation to microscaled 4-bit floating point, and back.
//
// A warp takes 512 columns of one row: 32 groups of 16, one per lane (an
// nvfp4 block; half an mxfp4 block, whose two lanes share their maximum). A
// CTA's eight warps take rows 2i, 2i + 1 of the four 32-row quarters of a
// scale tile: those rows' scales share 32-byte sectors. Rows whose addresses
// allow it are read with 16-byte loads; the others element by element,
// coalesced, through shared memory. Bound by DRAM traffic: x is read once
// (twice when the tensor's scale is sought, the second time from the end, so
// that what the first pass left in L2 is found there), 0.5625 (0.53) bytes an
// element are written.
//
// Every rounding is spelled out (a reciprocal and products rounded to fp32,
// two conversions to nearest even), so codes are reproducible bit for bit
// from the formulas.
#include <algorithm>

#include "fp4.cuh"

namespace ts {
namespace fp4 {

constexpr int kWarps = 8;
constexpr int kSeg = 512;          // columns of a warp's piece
constexpr int kMaxParts = 1184;    // CTAs of the maximum pass

struct QuantArgs {
  const void* x;
  int64_t rows, cols, stride;   // stride in elements
  uint8_t* codes;
  uint8_t* scales;
  float* global_scale;
  int64_t row_bytes, kt;        // bytes of a row of codes, scale tiles along a row
  int segs;
  int reverse;                  // walk from the end
  uint32_t* parts;              // bits of the CTAs' maxima when the scale is sought, else NULL
  int n_parts;
};

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

// 16 elements of a row from column c0 on (zeros behind the last column).
// ALIGNED: the row starts on a 16-byte boundary (c0 is a multiple of 16).
// Otherwise the warp stages its 512 columns in `stage`.
template <int DT, bool ALIGNED>
__device__ __forceinline__ void load16(const QuantArgs& a, int64_t row, int seg, int lane, typename Elem<DT>::T* stage,
                                       typename Elem<DT>::T (&v)[16]) {
  using T = typename Elem<DT>::T;
  const T* p = reinterpret_cast<const T*>(a.x) + row * a.stride;
  const int64_t first = (int64_t)seg * kSeg;
  if (ALIGNED) {
    const int64_t c0 = first + lane * 16;
    if (c0 + 16 <= a.cols) {
      constexpr int N = 16 * sizeof(T) / 16;
      uint4 w[N];
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint4*>(p + c0)[i];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = reinterpret_cast<const T*>(w)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = c0 + i < a.cols ? p[c0 + i] : (T)0;
    }
  } else {
    T t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int64_t c = first + i * 32 + lane;
      t[i] = c < a.cols ? p[c] : (T)0;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; ++i) stage[i * 32 + lane] = t[i];
    __syncwarp();
    constexpr int N = 16 * sizeof(T) / 16;
    uint4 w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint4*>(stage + lane * 16)[i];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = reinterpret_cast<const T*>(w)[i];
  }
}

// Largest magnitude as the type's bits (a NaN or infinity: at least kInf).
template <int DT>
__device__ __forceinline__ uint32_t top_bits(const typename Elem<DT>::T (&v)[16]) {
  constexpr uint32_t kAbs = DT == TS_F32 ? 0x7FFFFFFFu : 0x7FFFu;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, (uint32_t)v[i] & kAbs);
  return m;
}

template <int DT, bool ALIGNED>
__global__ void __launch_bounds__(kWarps * 32) fp4_amax_kernel(const QuantArgs a) {
  using E = Elem<DT>;
  __shared__ __align__(16) typename E::T stage[ALIGNED ? 1 : kWarps][ALIGNED ? 16 : kSeg];
  __shared__ uint32_t part[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t units = a.rows * a.segs;
  float m = 0.f;
  for (int64_t u = (int64_t)blockIdx.x * kWarps + warp; u < units; u += (int64_t)gridDim.x * kWarps) {
    typename E::T v[16];
    load16<DT, ALIGNED>(a, u / a.segs, (int)(u % a.segs), lane, stage[ALIGNED ? 0 : warp], v);
    if (top_bits<DT>(v) < E::kInf) {
      m = fmaxf(m, E::f((typename E::T)top_bits<DT>(v)));
    } else {   // only finite elements count
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float f = fabsf(E::f(v[i]));
        if (f < INFINITY) m = fmaxf(m, f);
      }
    }
  }
  const uint32_t w = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
  if (lane == 0) part[warp] = w;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) r = max(r, part[i]);
    a.parts[blockIdx.x] = r;
  }
}

template <int DT, bool NV, bool ALIGNED>
__global__ void __launch_bounds__(kWarps * 32) fp4_quantize_kernel(const QuantArgs a) {
  using E = Elem<DT>;
  __shared__ __align__(16) typename E::T stage[ALIGNED ? 1 : kWarps][ALIGNED ? 16 : kSeg];
  __shared__ uint32_t part[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float g = 1.f, to_scale = 0.f;
  if (NV) {
    if (a.parts != nullptr) {
      uint32_t w = 0;
      for (int i = threadIdx.x; i < a.n_parts; i += kWarps * 32) w = max(w, a.parts[i]);
      w = __reduce_max_sync(0xffffffffu, w);
      if (lane == 0) part[warp] = w;
      __syncthreads();
      w = 0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) w = max(w, part[i]);
      g = fmaxf(__fmul_rn(__uint_as_float(w), 1.f / 2688.f), kMinScale);   // 2688 = 448 * 6
      if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.global_scale = g;
    } else {
      g = usable_scale(a.global_scale);
    }
    to_scale = __frcp_rn(__fmul_rn(6.f, g));
  }
  const int bx = a.reverse ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const int64_t row = (int64_t)(bx >> 4) * kTileRows + (bx & 15) * 2 + (warp & 1) + (warp >> 1) * 32;
  if (row >= a.rows) return;
  for (int s = blockIdx.y; s < a.segs; s += gridDim.y) {
    const int seg = a.reverse ? a.segs - 1 - s : s;
    typename E::T v[16];
    load16<DT, ALIGNED>(a, row, seg, lane, stage[ALIGNED ? 0 : warp], v);
    uint32_t top = top_bits<DT>(v);
    if (!NV) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const bool bad = top >= E::kInf;
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
    uint2 out = make_uint2(0, 0);
    if (bad) {
      sc = NV ? 0x7Fu : 0xFFu;
    } else {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = E::f(v[i]);
      out.x = to_e2m1x8(f, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = E::f(v[8 + i]);
      out.y = to_e2m1x8(f, r);
    }
    const int64_t group = (int64_t)seg * 32 + lane;   // of 16 columns
    if (group * 8 < a.row_bytes) {
      *reinterpret_cast<uint2*>(a.codes + row * a.row_bytes + group * 8) = out;
      if (NV) a.scales[scale_at(row, group, a.kt)] = (uint8_t)sc;
      else if ((lane & 1) == 0) a.scales[scale_at(row, group >> 1, a.kt)] = (uint8_t)sc;
    }
  }
}

struct DequantArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  const float* global_scale;
  int64_t rows, cols, row_bytes, kt, out_stride;
  void* out;
  int segs;
};

template <int DT, bool NV, bool ALIGNED>
__global__ void __launch_bounds__(kWarps * 32) fp4_dequantize_kernel(const DequantArgs a) {
  using T = typename Elem<DT>::T;
  __shared__ __align__(16) T stage[ALIGNED ? 1 : kWarps][ALIGNED ? 16 : kSeg];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float g = NV ? usable_scale(a.global_scale) : 1.f;
  const int64_t row = (int64_t)(blockIdx.x >> 4) * kTileRows + (blockIdx.x & 15) * 2 + (warp & 1) + (warp >> 1) * 32;
  if (row >= a.rows) return;
  for (int seg = blockIdx.y; seg < a.segs; seg += gridDim.y) {
    const int64_t group = (int64_t)seg * 32 + lane;
    __align__(16) T v[16];
    if (group * 8 < a.row_bytes) {
      const uint2 w = *reinterpret_cast<const uint2*>(a.codes + row * a.row_bytes + group * 8);
      const uint8_t sb = a.scales[scale_at(row, NV ? group : group >> 1, a.kt)];
      const float s = NV ? __fmul_rn(e4m3_value(sb), g) : e8m0_value(sb);
      uint32_t h[8];
      uint32_t (&h0)[4] = *reinterpret_cast<uint32_t(*)[4]>(h);
      uint32_t (&h1)[4] = *reinterpret_cast<uint32_t(*)[4]>(h + 4);
      from_e2m1x8(w.x, h0);
      from_e2m1x8(w.y, h1);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        const float y0 = __fmul_rn(f.x, s), y1 = __fmul_rn(f.y, s);
        if (DT == TS_F32) {
          v[2 * i] = (T)__float_as_uint(y0);
          v[2 * i + 1] = (T)__float_as_uint(y1);
        } else if (DT == TS_BF16) {
          v[2 * i] = (T)__bfloat16_as_ushort(__float2bfloat16_rn(y0));
          v[2 * i + 1] = (T)__bfloat16_as_ushort(__float2bfloat16_rn(y1));
        } else {
          v[2 * i] = (T)__half_as_ushort(__float2half_rn(y0));
          v[2 * i + 1] = (T)__half_as_ushort(__float2half_rn(y1));
        }
      }
    }
    T* p = reinterpret_cast<T*>(a.out) + row * a.out_stride;
    const int64_t c0 = group * 16;
    if (ALIGNED) {
      if (c0 + 16 <= a.cols) {
#pragma unroll
        for (int i = 0; i < (int)(16 * sizeof(T) / 16); ++i)
          reinterpret_cast<uint4*>(p + c0)[i] = reinterpret_cast<const uint4*>(v)[i];
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c0 + i < a.cols) p[c0 + i] = v[i];
      }
    } else {
      T* st = stage[warp];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < (int)(16 * sizeof(T) / 16); ++i)
        reinterpret_cast<uint4*>(st + lane * 16)[i] = reinterpret_cast<const uint4*>(v)[i];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int64_t c = (int64_t)seg * kSeg + i * 32 + lane;
        if (c < a.cols) p[c] = st[i * 32 + lane];
      }
    }
  }
}

int check_tensor(const ts_fp4_tensor* t, const char* what) {
  TS_REQUIRE(t != nullptr, "%s: NULL tensor", what);
  TS_UNSUPPORTED(t->format == TS_NVFP4 || t->format == TS_MXFP4, "%s: unknown format %d", what, (int)t->format);
  TS_REQUIRE(t->rows >= 0 && t->cols > 0, "%s: bad shape", what);
  TS_UNSUPPORTED(t->rows < ((int64_t)1 << 31) - 128 && t->cols < ((int64_t)1 << 31) - 64, "%s: too large", what);
  TS_REQUIRE(t->rows == 0 || (t->codes && t->scales), "%s: NULL pointer", what);
  TS_REQUIRE(is_aligned(t->codes, 16) && is_aligned(t->scales, 16), "%s: codes and scales must be 16-byte aligned", what);
  return TS_OK;
}

// Grid of the row-tile kernels: 16 CTAs per 128 rows, enough along the
// columns to give every SM eight CTAs.
static dim3 tile_grid(int64_t rows, int segs) {
  const int64_t gx = (rows + kTileRows - 1) / kTileRows * 16;
  const int64_t want = ((int64_t)sm_count() * 16 + gx - 1) / gx;
  return dim3((unsigned)gx, (unsigned)std::min<int64_t>(segs, std::max<int64_t>(1, std::min<int64_t>(want, 65535))));
}

template <int DT, bool AL>
static int launch_quantize(const QuantArgs& a, bool nv, cudaStream_t st) {
  const dim3 grid = tile_grid(a.rows, a.segs);
  if (a.parts != nullptr) {
    fp4_amax_kernel<DT, AL><<<a.n_parts, kWarps * 32, 0, st>>>(a);
    TS_LAUNCH_CHECK();
  }
  if (nv) fp4_quantize_kernel<DT, true, AL><<<grid, kWarps * 32, 0, st>>>(a);
  else fp4_quantize_kernel<DT, false, AL><<<grid, kWarps * 32, 0, st>>>(a);
  TS_LAUNCH_CHECK();
  return TS_OK;
}

template <int DT, bool AL>
static int launch_dequantize(const DequantArgs& a, bool nv, cudaStream_t st) {
  const dim3 grid = tile_grid(a.rows, a.segs);
  if (nv) fp4_dequantize_kernel<DT, true, AL><<<grid, kWarps * 32, 0, st>>>(a);
  else fp4_dequantize_kernel<DT, false, AL><<<grid, kWarps * 32, 0, st>>>(a);
  TS_LAUNCH_CHECK();
  return TS_OK;
}

}  // namespace fp4
}  // namespace ts

using namespace ts;
using namespace ts::fp4;

extern "C" size_t ts_fp4_scales_bytes(int64_t rows, int64_t cols, int format) {
  if (rows < 0 || cols <= 0) return 0;
  return (size_t)((rows + kTileRows - 1) / kTileRows) * scale_tiles(cols, format) * kTileBytes;
}

extern "C" size_t ts_fp4_quantize_workspace_size(void) { return (size_t)kMaxParts * 4; }

extern "C" int ts_fp4_quantize(const void* x, int x_dtype, int64_t x_row_stride, const ts_fp4_tensor* t, int find_scale,
                               void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_tensor(t, "ts_fp4_quantize");
  if (rc != TS_OK) return rc;
  TS_UNSUPPORTED(x_dtype == TS_F16 || x_dtype == TS_BF16 || x_dtype == TS_F32, "unknown element type %d", x_dtype);
  const bool nv = t->format == TS_NVFP4;
  TS_REQUIRE(!find_scale || (nv && t->global_scale), "only an nvfp4 tensor with a global_scale has one to find");
  if (t->rows == 0) return TS_OK;
  TS_REQUIRE(x, "NULL pointer");
  if (find_scale && (workspace == nullptr || workspace_bytes < ts_fp4_quantize_workspace_size())) {
    set_error("workspace of %zu bytes, %zu needed", workspace_bytes, ts_fp4_quantize_workspace_size());
    return TS_ERR_WORKSPACE;
  }
  QuantArgs a;
  a.x = x;
  a.rows = t->rows;
  a.cols = t->cols;
  a.stride = x_row_stride;
  a.codes = t->codes;
  a.scales = t->scales;
  a.global_scale = t->global_scale;
  a.row_bytes = padded_cols(t->cols) / 2;
  a.kt = scale_tiles(t->cols, t->format);
  a.segs = (int)((padded_cols(t->cols) + kSeg - 1) / kSeg);
  a.reverse = find_scale ? 1 : 0;
  a.parts = find_scale ? reinterpret_cast<uint32_t*>(workspace) : nullptr;
  a.n_parts = (int)std::min<int64_t>(std::min(kMaxParts, sm_count() * 4), (a.rows * a.segs + kWarps - 1) / kWarps);
  const int es = x_dtype == TS_F32 ? 4 : 2;
  const bool al = is_aligned(x, 16) && (x_row_stride * es) % 16 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (x_dtype == TS_F16) return al ? launch_quantize<TS_F16, true>(a, nv, st) : launch_quantize<TS_F16, false>(a, nv, st);
  if (x_dtype == TS_BF16)
    return al ? launch_quantize<TS_BF16, true>(a, nv, st) : launch_quantize<TS_BF16, false>(a, nv, st);
  return al ? launch_quantize<TS_F32, true>(a, nv, st) : launch_quantize<TS_F32, false>(a, nv, st);
}

extern "C" int ts_fp4_dequantize(const ts_fp4_tensor* t, void* out, int out_dtype, int64_t out_row_stride,
                                 void* stream) {
  const int rc = check_tensor(t, "ts_fp4_dequantize");
  if (rc != TS_OK) return rc;
  TS_UNSUPPORTED(out_dtype == TS_F16 || out_dtype == TS_BF16 || out_dtype == TS_F32, "unknown element type %d",
                 out_dtype);
  if (t->rows == 0) return TS_OK;
  TS_REQUIRE(out, "NULL pointer");
  DequantArgs a;
  a.codes = t->codes;
  a.scales = t->scales;
  a.global_scale = t->global_scale;
  a.rows = t->rows;
  a.cols = t->cols;
  a.row_bytes = padded_cols(t->cols) / 2;
  a.kt = scale_tiles(t->cols, t->format);
  a.out_stride = out_row_stride;
  a.out = out;
  a.segs = (int)((t->cols + kSeg - 1) / kSeg);
  const bool nv = t->format == TS_NVFP4;
  const int es = out_dtype == TS_F32 ? 4 : 2;
  const bool al = is_aligned(out, 16) && (out_row_stride * es) % 16 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (out_dtype == TS_F16)
    return al ? launch_dequantize<TS_F16, true>(a, nv, st) : launch_dequantize<TS_F16, false>(a, nv, st);
  if (out_dtype == TS_BF16)
    return al ? launch_dequantize<TS_BF16, true>(a, nv, st) : launch_dequantize<TS_BF16, false>(a, nv, st);
  return al ? launch_dequantize<TS_F32, true>(a, nv, st) : launch_dequantize<TS_F32, false>(a, nv, st);
}
