// Quantisation of rows to 8-bit integers, and back.
//
//   s_r = max(max|x_r| / 127, 2^-100),   q = rint(x / s_r)
//
// with the quotients as products: s = max|x| * fp32(1 / 127) and x * (1 / s), every
// operation rounded to fp32. A row that holds an infinity or a NaN has the scale
// NaN and codes of 0, so that its values come back as NaN.
//
// A group of threads takes a row, eight neighbouring columns a thread and step,
// and keeps it in registers between the maximum and the codes, so that x is
// read once: up to 32 columns a thread, groups of a warp to a CTA of 1024 threads;
// rows of more than 32768 columns are read a second time, from L2. Rows that do
// not start on 16 bytes are read in words, shifted where they start in the
// middle of one. Bound by DRAM traffic: 8191 x 8192 bf16 33 to 35 us, 5.8 to 6.0 TB/s; one row of
// 4096, 2.0 us.
#include <algorithm>

#include "int8.cuh"

namespace ts {
namespace int8 {

constexpr int kHold = 4;           // chunks of eight columns that a thread keeps

struct QuantArgs {
  const void* x;
  int64_t rows, cols, stride;
  int8_t* codes;
  int64_t ld;
  float* scales;
  int chunks;                      // of a row, its padding to 16 columns included
};

// G: threads of a row (a warp to 1024); rows of more than kHold * G chunks are read twice.
template <int DT, bool AL, int G>
__global__ void __launch_bounds__(G < 256 ? 256 : G) int8_quantize_kernel(const QuantArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int kThreads = G < 256 ? 256 : G, N = DT == TS_F32 ? 8 : 4;
  __shared__ uint32_t tops[kThreads / 32];
  pdl_launch_dependents();                             // the product loads its weights meanwhile
  const int t = threadIdx.x % G, warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
  const bool has = row < a.rows;
  const T* x = reinterpret_cast<const T*>(a.x) + (has ? row * a.stride : 0);
  const int64_t cols = has ? a.cols : 0;
  uint32_t w[kHold][N];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kHold; ++i) load8<DT, AL>(x, t + i * G, cols, w[i]);
#pragma unroll
  for (int i = 0; i < kHold; ++i) top = max(top, top8<DT>(w[i]));
  for (int c = t + kHold * G; c < a.chunks; c += G) {
    uint32_t v[N];
    load8<DT, AL>(x, c, cols, v);
    top = max(top, top8<DT>(v));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (G > 32) {
    if ((threadIdx.x & 31) == 0) tops[warp] = top;
    __syncthreads();
    const int w0 = threadIdx.x / G * (G / 32);
#pragma unroll
    for (int i = 0; i < G / 32; ++i) top = max(top, tops[w0 + i]);
  }
  if (!has) return;
  const bool finite = top < 0x7F800000u;
  const float s = finite ? scale_of(__uint_as_float(top)) : __uint_as_float(0x7FC00000u);
  const float r = finite ? __frcp_rn(s) : 0.f;
  if (t == 0) a.scales[row] = s;
  int8_t* out = a.codes + row * a.ld;
#pragma unroll
  for (int i = 0; i < kHold; ++i) {
    const int c = t + i * G;
    if (c < a.chunks) *reinterpret_cast<uint2*>(out + 8 * (int64_t)c) = finite ? codes8<DT>(w[i], r) : make_uint2(0, 0);
  }
  for (int c = t + kHold * G; c < a.chunks; c += G) {
    uint32_t v[N];
    load8<DT, AL>(x, c, cols, v);
    *reinterpret_cast<uint2*>(out + 8 * (int64_t)c) = finite ? codes8<DT>(v, r) : make_uint2(0, 0);
  }
}

// The values q s of the first `cols` columns, a thread eight of them. 14336 x 4096 to bf16 50 us, 3.5 TB/s (27 us at the
// copy's bandwidth), to fp32 79, 3.7 TB/s (45): every eight values take a 64-bit division and the choice of the type.
__global__ void __launch_bounds__(256) int8_dequantize_kernel(const int8_t* codes, int64_t ld, const float* scales, int64_t rows,
                                                              int64_t cols, void* out, int dtype, int64_t out_stride, int vec) {
  const int64_t chunks = (cols + 7) / 8;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < rows * chunks; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / chunks, c = i - row * chunks;
    const uint2 q = *reinterpret_cast<const uint2*>(codes + row * ld + 8 * c);
    const float s = scales[row];
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __fmul_rn((float)(int8_t)((e < 4 ? q.x : q.y) >> (8 * (e & 3))), s);
    const int64_t at = row * out_stride + 8 * c;
    const int n = (int)min((int64_t)8, cols - 8 * c);
    if (vec && n == 8) {
      if (dtype == TS_F32) {
        float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at);
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        uint32_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (dtype == TS_BF16) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
            h[e] = *reinterpret_cast<const uint32_t*>(&b);
          } else {
            const __half2 b = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
            h[e] = *reinterpret_cast<const uint32_t*>(&b);
          }
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + at) = make_uint4(h[0], h[1], h[2], h[3]);
      }
    } else {
      for (int e = 0; e < n; ++e) store_f(out, dtype, at + e, v[e]);
    }
  }
}

template <int DT, bool AL>
static void launch_quantize(const QuantArgs& a, cudaStream_t st) {
  auto run = [&](auto k, int group) {
    const int per = group < 256 ? 256 / group : 1;
    k<<<(unsigned)((a.rows + per - 1) / per), std::max(group, 256), 0, st>>>(a);
  };
  // the smallest group that keeps a row in registers
  if (a.chunks <= kHold * 32) run(int8_quantize_kernel<DT, AL, 32>, 32);
  else if (a.chunks <= kHold * 128) run(int8_quantize_kernel<DT, AL, 128>, 128);
  else if (a.chunks <= kHold * 256) run(int8_quantize_kernel<DT, AL, 256>, 256);
  else if (a.chunks <= kHold * 512) run(int8_quantize_kernel<DT, AL, 512>, 512);
  else run(int8_quantize_kernel<DT, AL, 1024>, 1024);
}

int check_tensor(const ts_int8_tensor* t, const char* what) {
  TS_REQUIRE(t != nullptr, "%s: NULL tensor", what);
  TS_REQUIRE(t->rows >= 0 && t->cols > 0, "%s: bad shape", what);
  TS_REQUIRE(t->rows == 0 || (t->codes && t->scales), "%s: NULL pointer", what);
  TS_REQUIRE(t->row_stride % 16 == 0 && t->row_stride >= padded_cols(t->cols) && is_aligned(t->codes, 16),
             "%s: rows of codes must start on 16 bytes and be padded to 16 columns", what);
  TS_REQUIRE(is_aligned(t->scales, 4), "%s: scales must be aligned", what);
  // the sum of K products of codes stays within 32 bits
  TS_UNSUPPORTED(t->cols <= kMaxCols, "%s: more than %lld columns", what, (long long)kMaxCols);
  TS_UNSUPPORTED(t->rows < (int64_t)1 << 31, "%s: too many rows", what);
  return TS_OK;
}

}  // namespace int8
}  // namespace ts

using namespace ts;
using namespace ts::int8;

extern "C" int ts_int8_quantize(const void* x, int x_dtype, int64_t x_row_stride, const ts_int8_tensor* t, void* stream) {
  const int rc = check_tensor(t, "ts_int8_quantize");
  if (rc != TS_OK) return rc;
  TS_UNSUPPORTED(x_dtype == TS_F16 || x_dtype == TS_BF16 || x_dtype == TS_F32, "unknown element type %d", x_dtype);
  if (t->rows == 0) return TS_OK;
  const int size = x_dtype == TS_F32 ? 4 : 2;
  TS_REQUIRE(x && is_aligned(x, size), "x must be aligned to its elements");
  QuantArgs a;
  a.x = x;
  a.rows = t->rows;
  a.cols = t->cols;
  a.stride = x_row_stride;
  a.codes = t->codes;
  a.ld = t->row_stride;
  a.scales = t->scales;
  a.chunks = (int)(padded_cols(t->cols) / 8);
  const bool al = is_aligned(x, 16) && (x_row_stride * size) % 16 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (x_dtype == TS_BF16) al ? launch_quantize<TS_BF16, true>(a, st) : launch_quantize<TS_BF16, false>(a, st);
  else if (x_dtype == TS_F16) al ? launch_quantize<TS_F16, true>(a, st) : launch_quantize<TS_F16, false>(a, st);
  else al ? launch_quantize<TS_F32, true>(a, st) : launch_quantize<TS_F32, false>(a, st);
  TS_LAUNCH_CHECK();
  return TS_OK;
}

extern "C" int ts_int8_dequantize(const ts_int8_tensor* t, void* out, int out_dtype, int64_t out_row_stride, void* stream) {
  const int rc = check_tensor(t, "ts_int8_dequantize");
  if (rc != TS_OK) return rc;
  TS_UNSUPPORTED(out_dtype == TS_F16 || out_dtype == TS_BF16 || out_dtype == TS_F32, "unknown output type %d", out_dtype);
  if (t->rows == 0) return TS_OK;
  TS_REQUIRE(out, "NULL pointer");
  const int64_t items = t->rows * ((t->cols + 7) / 8);
  const int vec = is_aligned(out, 16) && out_row_stride % 8 == 0;
  const unsigned grid = (unsigned)std::min<int64_t>((items + 255) / 256, (int64_t)sm_count() * 32);
  int8_dequantize_kernel<<<grid, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      t->codes, t->row_stride, t->scales, t->rows, t->cols, out, out_dtype, out_row_stride, vec);
  TS_LAUNCH_CHECK();
  return TS_OK;
}
