// Quantisation to microscaled 4-bit floating point, and back.
//
// A warp takes 128 columns of the four rows that share 16-byte units of a scale
// tile (r, r + 32, r + 64, r + 96): 16 columns per lane, an nvfp4 block or half
// an mxfp4 block, whose two lanes share their maximum. A CTA's eight warps take
// eight neighbouring such rows, so that its scales are whole 128-byte lines.
// Rows that start on 32 or 16 bytes are read with loads that wide; the others
// word by word, coalesced, through shared memory. Bound by DRAM traffic: x is
// read once (twice when the tensor's scale is sought, the second time from the
// end, so that what the first pass left in L2 is found there), 0.5625 (0.53)
// bytes an element are written. Measured: 14336 x 4096 fp16, 27 us behind the
// maximum pass and 26 us back, 5.7 TB/s; 2047 x 14330 bf16 (rows that start in
// the middle of a word), 19 us and 15 us, 3.9 and 4.8 TB/s, bound by the words'
// way through shared memory; 1 x 4096, 2.0 us each.
//
// Every rounding is spelled out (a reciprocal and products rounded to fp32,
// two conversions to nearest even), so codes are reproducible bit for bit
// from the formulas.
#include <algorithm>

#include "fp4.cuh"
#include "gemm.cuh"
#include "paged.cuh"

namespace ts {
namespace fp4 {

constexpr int kWarps = 8;
constexpr int kAmaxSeg = 512;      // columns of a warp's piece of the maximum pass
constexpr int kSeg = 128;          // columns of a warp's piece, four rows high
constexpr int kAmaxUnits = 4;      // pieces that a warp of the maximum pass has in flight
constexpr int kSmallUnits = 4;     // pieces that a warp of the one-pass kernel keeps
constexpr int kSmallCtas = 8;      // CTAs (a cluster) of the one-pass kernel at most

struct QuantArgs {
  const void* x;
  int64_t rows, cols, stride;   // stride in elements
  uint8_t* codes;
  uint8_t* scales;
  float* global_scale;
  int64_t row_bytes, kt;        // bytes of a row of codes, scale tiles along a row
  int segs;
  int reverse;                  // walk from the end
  int64_t amax_cols;            // the maximum pass takes rows without gaps as one row
  int amax_rows, amax_segs;
  int groups;                   // groups of rows r, r + 32, r + 64, r + 96
  int* counters;                // CTAs that have left their maximum, the maximum's bits; zero between calls
};

// 32 bytes from a 32-byte boundary.
__device__ __forceinline__ void ld32(const void* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}
__device__ __forceinline__ void st32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Where a lane reads (or writes) its share of a warp's four rows, row0 + 32 q.
// AL: the alignment of rows. With 32 or 16, eight lanes take a row, 16
// consecutive columns each. With 4, all 32 lanes take one row after the other
// in words, and deal() sorts them. With 2 (16-bit elements) the four rows may
// start in the middle of a word: the words are then those behind the first
// element.
template <int DT, int AL>
struct Place {
  using T = typename Elem<DT>::T;
  const char* p;     // this lane's place in columns 0 .. 127
  int64_t step;      // bytes from one of the four rows to the next (AL < 16)
  int rows;          // of the four, how many exist (AL >= 16: whether this lane's does)
  int mid;           // the rows start in the middle of a word
  __device__ __forceinline__ Place(const void* x, int64_t n_rows, int64_t stride, int64_t row0, int lane) {
    const T* t = reinterpret_cast<const T*>(x);
    const int64_t left = n_rows - row0;
    mid = 0;
    if (AL >= 16) {
      p = reinterpret_cast<const char*>(t + (row0 + (lane >> 3) * 32) * stride + (lane & 7) * 16);
      rows = left > (lane >> 3) * 32;
    } else {
      const T* r = t + row0 * stride;
      if (AL == 2) mid = (int)(reinterpret_cast<uintptr_t>(r) >> 1) & 1;
      p = reinterpret_cast<const char*>(r + mid) + lane * 4;
      rows = left > 96 ? 4 : left > 64 ? 3 : left > 32 ? 2 : left > 0 ? 1 : 0;
    }
    step = stride * 32 * (int64_t)sizeof(T);
  }
};

// Reads columns [first, first + 128), of which `left` exist (zeros for the
// others and for rows that do not exist).
template <int DT, int AL>
__device__ __forceinline__ void load16(const Place<DT, AL>& w, int64_t first, int64_t left64, int lane, Lane<DT>& v) {
  using T = typename Elem<DT>::T;
  constexpr int N = Lane<DT>::N;
  const int left = (int)min((int64_t)kSeg + 1, left64);
  const char* p = w.p + first * (int)sizeof(T);
  v.e = 0;
  if (AL == 2 && w.mid && lane < w.rows && left > 0)
    v.e = *reinterpret_cast<const T*>(p - lane * 4 - 2 + lane * w.step);
  if (left >= kSeg + w.mid && (AL >= 16 ? w.rows : w.rows == 4)) {
    if constexpr (AL == 32) {
#pragma unroll
      for (int i = 0; i < N / 8; ++i) ld32(p + 32 * i, *reinterpret_cast<uint32_t(*)[8]>(v.w + 8 * i));
    } else if constexpr (AL == 16) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + i);
        v.w[4 * i] = u.x; v.w[4 * i + 1] = u.y; v.w[4 * i + 2] = u.z; v.w[4 * i + 3] = u.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        v.w[i] = __ldg(reinterpret_cast<const uint32_t*>(p + i / (N / 4) * w.step + i % (N / 4) * 128));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v.w[i] = 0;
  if constexpr (AL >= 16) {
    if (!w.rows) return;
    const T* t = reinterpret_cast<const T*>(p);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if ((lane & 7) * 16 + i < left) {
        if (DT == TS_F32) v.w[i % N] = (uint32_t)t[i];
        else v.w[(i / 2) % N] |= (uint32_t)t[i] << (16 * (i & 1));
      }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i / (N / 4) >= w.rows) break;
      const char* q = p + i / (N / 4) * w.step + i % (N / 4) * 128;
      const int word = i % (N / 4) * 32 + lane;
      if (DT == TS_F32) {
        if (word < left) v.w[i] = *reinterpret_cast<const uint32_t*>(q);
      } else {
        const T* t = reinterpret_cast<const T*>(q);
        const int c = 2 * word + w.mid;               // the word's columns: c, c + 1
        if (c < left) v.w[i] = (uint32_t)t[0];
        if (c + 1 < left) v.w[i] |= (uint32_t)t[1] << 16;
      }
    }
  }
}

// From the order that load16 read words in (AL < 16) to 16 consecutive columns
// per lane, through the warp's 4 rows of shared memory.
template <int DT, int AL>
__device__ __forceinline__ void deal(const Place<DT, AL>& place, uint32_t* stage, int lane, Lane<DT>& v) {
  if constexpr (AL >= 16) return;
  constexpr int N = Lane<DT>::N;
  __syncwarp();
  if (AL == 2 && place.mid) {
    uint16_t* s = reinterpret_cast<uint16_t*>(stage);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = 2 * (i % (N / 4) * 32 + lane) + 1, r = i / (N / 4) * kSeg;
      s[r + c] = (uint16_t)v.w[i];
      if (c + 1 < kSeg) s[r + c + 1] = (uint16_t)(v.w[i] >> 16);
    }
    if (lane < 4) s[lane * kSeg] = (uint16_t)v.e;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) stage[i * 32 + lane] = v.w[i];
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const uint4 u = reinterpret_cast<const uint4*>(stage + lane * N)[i];
    v.w[4 * i] = u.x; v.w[4 * i + 1] = u.y; v.w[4 * i + 2] = u.z; v.w[4 * i + 3] = u.w;
  }
}

// 512 columns of one row from `first` on, as words in any order (for maxima).
template <int DT, int AL>
__device__ __forceinline__ void load_flat(const void* x, int64_t cols, int64_t row_at, int64_t first, int lane,
                                          Lane<DT>& v) {
  using T = typename Elem<DT>::T;
  constexpr int N = Lane<DT>::N;
  const T* p = reinterpret_cast<const T*>(x) + row_at;
#pragma unroll
  for (int i = 0; i < N; ++i) v.w[i] = 0;
  if (AL >= 16 && first + kAmaxSeg <= cols) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p + first) + i * 32 + lane);
      v.w[4 * i] = u.x; v.w[4 * i + 1] = u.y; v.w[4 * i + 2] = u.z; v.w[4 * i + 3] = u.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int word = i * 32 + lane;
    if (DT == TS_F32) {
      if (first + word < cols) v.w[i] = (uint32_t)p[first + word];
    } else {
      const int64_t c = first + word * 2;
      if (AL >= 4 && c + 1 < cols) v.w[i] = __ldg(reinterpret_cast<const uint32_t*>(p + c));
      else if (c < cols) v.w[i] = (uint32_t)p[c] | (c + 1 < cols ? (uint32_t)p[c + 1] << 16 : 0);
    }
  }
}

// The largest finite magnitude.
template <int DT>
__device__ __forceinline__ float top_finite(const Lane<DT>& v) {
  using E = Elem<DT>;
  const uint32_t top = top_bits<DT>(v);
  if (top < E::kInf) return E::f((typename E::T)top);
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float f = fabsf(elem<DT>(v, i));
    if (f < INFINITY) m = fmaxf(m, f);
  }
  return m;
}

// The tensor's scale for a largest magnitude of `top`; 2688 = 448 * 6.
__device__ __forceinline__ float scale_for(float top) { return fmaxf(__fmul_rn(top, 1.f / 2688.f), kMinScale); }

// The tensor's scale. CTAs take the maximum in the workspace (its order does
// not matter); the last to arrive finishes it. 14336 x 4096 fp16, launch
// included: 25.6 us (30.1 us with a maximum per CTA that the last one gathers
// behind fences).
template <int DT, int AL>
__global__ void __launch_bounds__(kWarps * 32) fp4_amax_kernel(const QuantArgs a) {
  __shared__ uint32_t part[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // a warp takes 512 columns of a row: four "rows" of 128, one behind the other
  const int step = gridDim.x * kWarps, units = a.amax_rows * a.amax_segs;
  float m = 0.f;
  for (int u = blockIdx.x * kWarps + warp; u < units; u += kAmaxUnits * step) {
    Lane<DT> v[kAmaxUnits];
#pragma unroll
    for (int k = 0; k < kAmaxUnits; ++k) {
      const int w = u + k * step, row = a.amax_rows == 1 ? 0 : w / a.amax_segs;
      load_flat<DT, AL>(a.x, w < units ? a.amax_cols : 0, row * a.stride, (int64_t)(w - row * a.amax_segs) * kAmaxSeg, lane,
                        v[k]);
    }
#pragma unroll
    for (int k = 0; k < kAmaxUnits; ++k) m = fmaxf(m, top_finite<DT>(v[k]));
  }
  const uint32_t w = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
  if (lane == 0) part[warp] = w;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) r = max(r, part[i]);
    asm volatile("red.relaxed.gpu.global.max.u32 [%0], %1;" ::"l"(a.counters + 1), "r"(r) : "memory");
    int seen;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(seen) : "l"(a.counters) : "memory");
    if (seen == (int)gridDim.x - 1) {
      const float top = __uint_as_float((uint32_t)__ldcg(a.counters + 1));
      a.counters[0] = a.counters[1] = 0;
      *a.global_scale = scale_for(top);
    }
  }
}

template <int DT, bool NV, int AL>
__global__ void __launch_bounds__(kWarps * 32, DT == TS_F32 ? 6 : 7) fp4_quantize_kernel(const QuantArgs a) {
  __shared__ __align__(16) uint32_t stage[AL >= 16 ? 1 : kWarps][AL >= 16 ? 4 : 32 * Lane<DT>::N];
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float g = NV ? usable_scale(a.global_scale) : 1.f;
  const float to_scale = NV ? __frcp_rn(__fmul_rn(6.f, g)) : 0.f;
  const int bx = a.reverse ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const int64_t row0 = (int64_t)(bx >> 2) * kTileRows + (bx & 3) * 8 + warp, row = row0 + (lane >> 3) * 32;
  if (row0 >= a.rows) return;
  const bool exists = row < a.rows;
  const Place<DT, AL> src(a.x, a.rows, a.stride, row0, lane);
  uint8_t* codes = a.codes + row * a.row_bytes + (lane & 7) * 8;
  uint8_t* scales = a.scales + scale_at(row, NV ? lane & 7 : (lane & 7) >> 1, a.kt);
  const int groups = (int)(a.row_bytes / 8);             // of 16 columns
  for (int s = blockIdx.y; s < a.segs; s += gridDim.y) {
    const int seg = a.reverse ? a.segs - 1 - s : s;
    Lane<DT> v;
    load16<DT, AL>(src, (int64_t)seg * kSeg, a.cols - (int64_t)seg * kSeg, lane, v);
    deal<DT, AL>(src, stage[AL >= 16 ? 0 : warp], lane, v);
    uint2 out;
    const uint32_t sc = quantise16<DT, NV>(v, g, to_scale, out);
    if (exists && seg * 8 + (lane & 7) < groups) {
      *reinterpret_cast<uint2*>(codes + (int64_t)seg * 64) = out;
      // 128 columns are two scale tiles of nvfp4, one of mxfp4
      if (NV || (lane & 1) == 0) scales[(int64_t)seg * (NV ? 2 : 1) * kTileBytes] = (uint8_t)sc;
    }
  }
}

// A tensor of few pieces, its scale included, in one pass of one cluster: the
// pieces stay in registers while the CTAs tell one another their maxima.
// 8 x 4096 bf16: 4.8 us on the device, 8.5 us a call (9 x 4096, by the maximum
// pass and the quantiser: 5.8 and 11.8 us); 1 x 4096: 2.8 us.
template <int DT, int AL>
__global__ void __launch_bounds__(kWarps * 32) fp4_quantize_small_kernel(const QuantArgs a) {
  __shared__ __align__(16) uint32_t stage[AL >= 16 ? 1 : kWarps][AL >= 16 ? 4 : 32 * Lane<DT>::N];
  __shared__ uint32_t part[kWarps], mine;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, step = gridDim.x * kWarps;
  const int items = a.groups * a.segs, first = blockIdx.x * kWarps + warp;
  auto row0_of = [&](int group) { return (int64_t)(group >> 5) * kTileRows + (group & 31); };
  Lane<DT> v[kSmallUnits];
#pragma unroll
  for (int k = 0; k < kSmallUnits; ++k) {
    const int i = first + k * step, group = i / a.segs, seg = i - group * a.segs;
    const Place<DT, AL> src(a.x, i < items ? a.rows : 0, a.stride, i < items ? row0_of(group) : 0, lane);
    load16<DT, AL>(src, (int64_t)seg * kSeg, a.cols - (int64_t)seg * kSeg, lane, v[k]);
  }
  float m = 0.f;
#pragma unroll
  for (int k = 0; k < kSmallUnits; ++k) {
    const int i = first + k * step;
    if (i >= items) break;
    const Place<DT, AL> src(a.x, a.rows, a.stride, row0_of(i / a.segs), lane);
    deal<DT, AL>(src, stage[AL >= 16 ? 0 : warp], lane, v[k]);
    m = fmaxf(m, top_finite<DT>(v[k]));
  }
  const uint32_t w = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
  if (lane == 0) part[warp] = w;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) r = max(r, part[i]);
    mine = r;
  }
  __syncthreads();
  cluster_sync();
  uint32_t r = 0;
  if (lane < (int)gridDim.x)
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(r) : "r"(map_cta(smem_u32(&mine), lane)) : "memory");
  const float found = scale_for(__uint_as_float(__reduce_max_sync(0xffffffffu, r)));
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.global_scale = found;
  const float g = usable_scale(&found), to_scale = __frcp_rn(__fmul_rn(6.f, g));
#pragma unroll
  for (int k = 0; k < kSmallUnits; ++k) {
    const int i = first + k * step, group = i / a.segs, seg = i - group * a.segs;
    if (i >= items) break;
    const int64_t row = row0_of(group) + (lane >> 3) * 32;
    uint2 out;
    const uint32_t sc = quantise16<DT, true>(v[k], g, to_scale, out);
    if (row < a.rows && seg * 8 + (lane & 7) < (int)(a.row_bytes / 8)) {
      *reinterpret_cast<uint2*>(a.codes + row * a.row_bytes + (lane & 7) * 8 + (int64_t)seg * 64) = out;
      a.scales[scale_at(row, seg * 8 + (lane & 7), a.kt)] = (uint8_t)sc;
    }
  }
  cluster_sync();                                      // nobody leaves while its maximum may be read
}

struct DequantArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  const float* global_scale;
  int64_t rows, cols, row_bytes, kt, out_stride;
  void* out;
  int segs;
};

template <int DT, bool NV, int AL>
__global__ void __launch_bounds__(kWarps * 32, 7) fp4_dequantize_kernel(const DequantArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int N = Lane<DT>::N;
  __shared__ __align__(16) uint32_t stage[AL >= 16 ? 1 : kWarps][AL >= 16 ? 4 : 32 * N];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l8 = lane & 7;
  const float g = NV ? usable_scale(a.global_scale) : 1.f;
  const int64_t row0 = (int64_t)(blockIdx.x >> 2) * kTileRows + (blockIdx.x & 3) * 8 + warp, row = row0 + (lane >> 3) * 32;
  if (row0 >= a.rows) return;
  const bool exists = row < a.rows;
  const Place<DT, AL> dst(a.out, a.rows, a.out_stride, row0, lane);
  const uint8_t* codes = a.codes + row * a.row_bytes + l8 * 8;
  const uint8_t* scales = a.scales + scale_at(row, NV ? l8 : l8 >> 1, a.kt);
  const int groups = (int)(a.row_bytes / 8);             // of 16 columns
  for (int seg = blockIdx.y; seg < a.segs; seg += gridDim.y) {
    uint2 w = make_uint2(0, 0);
    uint8_t sb = 0;
    if (exists && seg * 8 + l8 < groups) {
      w = __ldg(reinterpret_cast<const uint2*>(codes + (int64_t)seg * 64));
      sb = __ldg(scales + (int64_t)seg * (NV ? 2 : 1) * kTileBytes);
    }
    const float s = NV ? __fmul_rn(e4m3_value(sb), g) : e8m0_value(sb);
    uint32_t h[8];
    from_e2m1x8(w.x, *reinterpret_cast<uint32_t(*)[4]>(h));
    from_e2m1x8(w.y, *reinterpret_cast<uint32_t(*)[4]>(h + 4));
    __align__(16) uint32_t v[N];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
      const float y0 = __fmul_rn(f.x, s), y1 = __fmul_rn(f.y, s);
      if (DT == TS_F32) {
        v[(2 * i) % N] = __float_as_uint(y0);
        v[(2 * i + 1) % N] = __float_as_uint(y1);
      } else if (DT == TS_BF16) {
        const __nv_bfloat162 b2 = __floats2bfloat162_rn(y0, y1);
        v[i] = *reinterpret_cast<const uint32_t*>(&b2);
      } else {
        const __half2 b2 = __floats2half2_rn(y0, y1);
        v[i] = *reinterpret_cast<const uint32_t*>(&b2);
      }
    }
    const int64_t first = (int64_t)seg * kSeg;
    const int left = (int)min((int64_t)kSeg, a.cols - first);
    char* p = const_cast<char*>(dst.p) + first * (int)sizeof(T);
    if constexpr (AL >= 16) {
      if (!dst.rows) continue;
      if (left == kSeg) {
        if constexpr (AL == 32) {
#pragma unroll
          for (int i = 0; i < N / 8; ++i) st32(p + 32 * i, v + 8 * i);
        } else {
#pragma unroll
          for (int i = 0; i < N / 4; ++i)
            reinterpret_cast<uint4*>(p)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (l8 * 16 + i < left)
            reinterpret_cast<T*>(p)[i] = DT == TS_F32 ? (T)v[i % N] : (T)(v[(i / 2) % N] >> (16 * (i & 1)));
      }
    } else {
      uint32_t* st = stage[warp];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < N / 4; ++i)
        reinterpret_cast<uint4*>(st + lane * N)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
      __syncwarp();
      if (AL == 2 && dst.mid) {
        // the first element of row `lane`, then the words behind it
        const uint16_t* h = reinterpret_cast<const uint16_t*>(st);
        if (lane < dst.rows) *reinterpret_cast<T*>(p - lane * 4 - 2 + lane * dst.step) = (T)h[lane * kSeg];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (i / (N / 4) >= dst.rows) break;
          char* q = p + i / (N / 4) * dst.step + i % (N / 4) * 128;
          const int c = 2 * (i % (N / 4) * 32 + lane) + 1, r = i / (N / 4) * kSeg;
          if (c + 1 < min(left, kSeg)) *reinterpret_cast<uint32_t*>(q) = (uint32_t)h[r + c] | ((uint32_t)h[r + c + 1] << 16);
          else if (c < left) *reinterpret_cast<T*>(q) = (T)h[r + c];
        }
        continue;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i / (N / 4) >= dst.rows) break;
        char* q = p + i / (N / 4) * dst.step + i % (N / 4) * 128;
        const uint32_t x = st[i * 32 + lane];
        const int word = i % (N / 4) * 32 + lane;
        if (left == kSeg) {
          *reinterpret_cast<uint32_t*>(q) = x;
        } else if (DT == TS_F32) {
          if (word < left) *reinterpret_cast<uint32_t*>(q) = x;
        } else {
          if (2 * word < left) reinterpret_cast<T*>(q)[0] = (T)x;
          if (2 * word + 1 < left) reinterpret_cast<T*>(q)[1] = (T)(x >> 16);
        }
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

// Grid of the row-tile kernels: 4 CTAs per 128 rows (one for up to 8) and
// enough along the columns for four waves of eight CTAs per SM. (Many short
// CTAs at full occupancy measured better than fewer with several pieces in
// flight each: 2047 x 14330, 18.6 against 20 to 32 us.)
static dim3 tile_grid(int64_t rows, int segs) {
  const int64_t gx = rows <= 8 ? 1 : (rows + kTileRows - 1) / kTileRows * 4;
  const int64_t want = ((int64_t)sm_count() * 32 + gx - 1) / gx;
  return dim3((unsigned)gx, (unsigned)std::min<int64_t>(segs, std::min<int64_t>(want, 65535)));
}

template <int DT, int AL>
static int launch_amax(const QuantArgs& a, cudaStream_t st) {
  const int64_t units = (int64_t)a.amax_rows * a.amax_segs;
  const int grid = (int)std::min<int64_t>(sm_count() * 3, (units + kWarps - 1) / kWarps);
  fp4_amax_kernel<DT, AL><<<grid, kWarps * 32, 0, st>>>(a);
  TS_LAUNCH_CHECK();
  return TS_OK;
}

template <int DT, int AL>
static int launch_small(const QuantArgs& a, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min(kSmallCtas, (a.groups * a.segs + kWarps - 1) / kWarps));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cfg.gridDim.x;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  TS_CUDA_TRY(cudaLaunchKernelEx(&cfg, fp4_quantize_small_kernel<DT, AL>, a));
  TS_LAUNCH_CHECK();
  return TS_OK;
}

template <int DT, int AL>
static int launch_quantize(const QuantArgs& a, bool nv, cudaStream_t st) {
  const dim3 grid = tile_grid(a.rows, a.segs);
  if (nv) fp4_quantize_kernel<DT, true, AL><<<grid, kWarps * 32, 0, st>>>(a);
  else fp4_quantize_kernel<DT, false, AL><<<grid, kWarps * 32, 0, st>>>(a);
  TS_LAUNCH_CHECK();
  return TS_OK;
}

template <int DT>
static int launch_quantize(const QuantArgs& a, int al, int amax_al, bool nv, bool find, cudaStream_t st) {
  if (find && (int64_t)a.groups * a.segs <= kSmallCtas * kWarps * kSmallUnits) {
    if (al == 32) return launch_small<DT, 32>(a, st);
    if (al == 16) return launch_small<DT, 16>(a, st);
    if (al == 4 || DT == TS_F32) return launch_small<DT, 4>(a, st);
    return launch_small<DT, DT == TS_F32 ? 4 : 2>(a, st);
  }
  if (find) {
    int rc;
    if (amax_al >= 16) rc = launch_amax<DT, 16>(a, st);
    else if (amax_al == 4 || DT == TS_F32) rc = launch_amax<DT, 4>(a, st);
    else rc = launch_amax<DT, DT == TS_F32 ? 4 : 2>(a, st);
    if (rc != TS_OK) return rc;
  }
  if (al == 32) return launch_quantize<DT, 32>(a, nv, st);
  if (al == 16) return launch_quantize<DT, 16>(a, nv, st);
  if (al == 4 || DT == TS_F32) return launch_quantize<DT, 4>(a, nv, st);
  return launch_quantize<DT, DT == TS_F32 ? 4 : 2>(a, nv, st);
}

template <int DT, int AL>
static int launch_dequantize(const DequantArgs& a, bool nv, cudaStream_t st) {
  const dim3 grid = tile_grid(a.rows, a.segs);
  if (nv) fp4_dequantize_kernel<DT, true, AL><<<grid, kWarps * 32, 0, st>>>(a);
  else fp4_dequantize_kernel<DT, false, AL><<<grid, kWarps * 32, 0, st>>>(a);
  TS_LAUNCH_CHECK();
  return TS_OK;
}

template <int DT>
static int launch_dequantize(const DequantArgs& a, int al, bool nv, cudaStream_t st) {
  if (al == 32) return launch_dequantize<DT, 32>(a, nv, st);
  if (al == 16) return launch_dequantize<DT, 16>(a, nv, st);
  if (al == 4 || DT == TS_F32) return launch_dequantize<DT, 4>(a, nv, st);
  return launch_dequantize<DT, DT == TS_F32 ? 4 : 2>(a, nv, st);
}

// Alignment of rows that the kernels use: 32, 16, 4 or 2 bytes.
static int row_alignment(const void* p, int64_t stride, int es) {
  for (int al : {32, 16, 4})
    if (is_aligned(p, al) && (stride * es) % al == 0) return al;
  return 2;
}

}  // namespace fp4
}  // namespace ts

using namespace ts;
using namespace ts::fp4;

extern "C" size_t ts_fp4_scales_bytes(int64_t rows, int64_t cols, int format) {
  if (rows < 0 || cols <= 0) return 0;
  return (size_t)((rows + kTileRows - 1) / kTileRows) * scale_tiles(cols, format) * kTileBytes;
}

extern "C" size_t ts_fp4_quantize_workspace_size(void) { return paged::kCounterBytes; }

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
  a.groups = (int)(t->rows / kTileRows * 32 + std::min<int64_t>(32, t->rows % kTileRows));
  a.counters = reinterpret_cast<int*>(workspace);
  const bool flat = x_row_stride == t->cols || t->rows == 1;
  a.amax_rows = flat ? 1 : (int)t->rows;
  a.amax_cols = flat ? t->rows * t->cols : t->cols;
  const int64_t amax_segs = (a.amax_cols + kAmaxSeg - 1) / kAmaxSeg;
  TS_UNSUPPORTED(!find_scale || a.amax_rows * amax_segs < ((int64_t)1 << 31) - (1 << 24), "tensor too large to find its scale");
  a.amax_segs = (int)amax_segs;
  const int es = x_dtype == TS_F32 ? 4 : 2, al = row_alignment(x, x_row_stride, es);
  const int amax_al = flat ? row_alignment(x, 0, es) : al;
  const bool find = find_scale != 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (x_dtype == TS_F16) return launch_quantize<TS_F16>(a, al, amax_al, nv, find, st);
  if (x_dtype == TS_BF16) return launch_quantize<TS_BF16>(a, al, amax_al, nv, find, st);
  return launch_quantize<TS_F32>(a, al, amax_al, nv, find, st);
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
  const int al = row_alignment(out, out_row_stride, out_dtype == TS_F32 ? 4 : 2);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (out_dtype == TS_F16) return launch_dequantize<TS_F16>(a, al, nv, st);
  if (out_dtype == TS_BF16) return launch_dequantize<TS_BF16>(a, al, nv, st);
  return launch_dequantize<TS_F32>(a, al, nv, st);
}
