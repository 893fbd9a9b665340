// Product of two microscaled 4-bit matrices on the block-scaled tensor cores.
//
//   out[m, n] = ga gb sum_k (qa sa)[m, k] (qb sb)[n, k] (+ bias[n])
//
// tcgen05.mma with block scaling multiplies E2M1 operands straight from
// shared memory and applies both blocks' scales from tensor memory inside the
// instruction, so neither operand is ever unpacked: K = 64 per instruction,
// one 32-bit TMEM column holding the four scales of a row (nvfp4; two of the
// four per instruction for mxfp4).
//
// Two kernels: fp4_gemm_kernel for decode-sized calls and small layers,
// fp4_pair_kernel (below) for prefill.
//
// fp4_gemm_kernel: a tile is 128 rows of b (the weight's output features; the
// MMA's M) x BT <= 128 rows of a (tokens; its N), K in stages of 256. Roles in
// one persistent CTA per SM:
//   warp 0      TMA producer: codes of both operands (128-byte rows, 128-byte
//               swizzle) and, as bulk copies, the scale tiles of the stage
//   warp 1      one thread copies the stage's scale tiles to TMEM
//               (tcgen05.cp, broadcast to the four lane quadrants) and issues
//               the stage's MMAs. Scales have TMEM columns per stage: a
//               stage's columns are rewritten only after the MMAs that read
//               them have released the stage.
//   warps 2-5   epilogue: tcgen05.ld, tensor scales, bias, stores
//   warps 6-13  (kernels of few tokens that come unquantised) quantise the
//               stage's tokens into shared memory, a stage per warp in turn
// Bound by the weight's bytes. The tiles are few, so they are split along K:
// into whole parts, whose CTAs are a cluster and add their sums through
// distributed shared memory, or, where clusters do not fit the tiles, into
// equal shares of all stages laid end to end, whose sums the last CTA of a
// tile to arrive adds from the workspace. Either way in CTA order. Measured, back
// to back in a graph: 14336 x 4096 nvfp4, 1 token 11.8 us, 128 tokens 14.4 (33 MB,
// 5.1 us at the copy bandwidth: 6.2 TB/s while the weight streams, the rest is
// start, first loads and epilogue); 4096 x 14336, four CTAs a tile, 33 tokens
// 13.8 us (15.8 by way of the workspace), 128 tokens 15.9 (19.0).
//
// Every wait is bounded in wall-clock time: a role whose wait runs out records
// a code and unwinds; the TMEM is freed at the end in any case.
#include <algorithm>

#include "fp4.cuh"
#include "paged.cuh"

namespace ts {
namespace fp4 {

constexpr int kBW = 128;                 // weight rows of a tile = TMEM lanes
constexpr int kBK = 256;                 // columns of a stage = one 128-byte row
constexpr int kEpiWarps = 4;
constexpr int kThreads = (2 + kEpiWarps) * 32;
constexpr int kQuantWarps = 8;

// Up to this many tokens the kernel quantises them itself, every CTA those of
// its stages; more come from a quantiser in front, which the kernel's start
// overlaps. nvfp4, 14336 x 4096, back to back in a graph: 1 token 11.3 us by
// itself, 8 tokens 12.4, 16 tokens 15.5; 9 to 16 tokens behind a quantiser 14.1.
constexpr int kOwnTokens = 8;
constexpr int kTmemCols = 512;
constexpr int kABytes = kBW * 128;
constexpr int kMaxCluster = 8;           // CTAs of a cluster that share a tile

__device__ int g_err;

struct GemmArgs {
  const uint8_t* wscales;
  const uint8_t* xscales;
  const float* wg;
  const float* xg;
  int64_t M, N;
  int wblocks, tblocks, kblocks;   // tiles of weight rows, of tokens, stages
  int kt, steps;                   // scale tiles along K, MMA steps of 64 columns
  const void* bias;
  int bias_dtype;
  void* out;
  int out_dtype;
  int64_t out_stride;
  int* counters;                   // one per tile, zero between calls
  float* partials;                 // [grid][2][BT / 4][128][4]
  uint64_t wait_ns;
  int stall;                       // test hook: the producer issues nothing
  int overlap;                     // launched while the quantisation of x may still run
  const void* x;                   // tokens to be quantised by the kernel itself
  int x_dtype, x_aligned;          // x_aligned: rows start on 16 bytes
  int64_t x_stride, K;
  int cluster;                     // CTAs that share a tile as a cluster, or 0
  int out_vec;                     // rows of out take stores of four values
};

template <bool NV, int BT>
struct Shape {
  static constexpr int kTiles = NV ? 4 : 2;                    // scale tiles of a stage, per 128 rows
  static constexpr int kSf = kTiles * kTileBytes;              // an operand's scales in a stage
  static constexpr int kXBytes = BT * 128;
  static constexpr int kStage = kABytes + kXBytes + 2 * kSf;
  static constexpr int kSfCols = 8 * kTiles;                   // TMEM columns of a stage's scales
  static constexpr int kAcc = 2;                               // accumulators
  static constexpr int kAccCols = BT < 32 ? 32 : BT;
  static constexpr int kFitTmem = (kTmemCols - kAcc * kAccCols) / kSfCols;
  static constexpr int kFitSmem = (227 * 1024 - 2048) / kStage;
  static constexpr int S = kFitTmem < kFitSmem ? (kFitTmem < 10 ? kFitTmem : 10) : (kFitSmem < 10 ? kFitSmem : 10);
  static constexpr size_t kSmem = 1024 + (size_t)S * kStage + (2 * S + 2 * kAcc + 1) * 8 + 16;
};

// A matrix descriptor of scale tiles: rows of 16 bytes, groups of eight rows
// 128 bytes apart, no swizzle.
__device__ __forceinline__ uint64_t desc_scales(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}

// 512 bytes of scales to four TMEM columns, in all four lane quadrants.
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

// Instruction descriptor: E2M1 operands, K-major, fp32 sums, M x N;
// sf: which of a column's scales the instruction starts from (mxfp4: 0 or 2).
template <bool NV>
__host__ __device__ constexpr uint32_t idesc_fp4(int M, int N, uint32_t sf) {
  return (sf << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (NV ? 0u : 1u << 23) |
         ((uint32_t)(M >> 7) << 27) | (sf << 29);
}

// One lane of a converged warp. Unlike `lane == 0` it tells the compiler that
// the code behind it runs once per warp, and the descriptors of tensor-core
// instructions then go to uniform registers without a loop over lanes (the
// same kernel, 8192 x 28672 x 8192: 2035 us with lane == 0, 1284 us with this).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}

template <bool NV>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                        uint32_t accumulate) {
  if (NV)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// Both tensor scales on a sum: as their product or, where that is no number of
// good precision, one after the other (the one that keeps clear of the range's end
// first), so that a result within the range is right for any pair of scales.
struct Alpha {
  float a, b;
  __device__ __forceinline__ Alpha(float x, float y) : a(x * y), b(1.f) {
    const bool high = a > 1.329227995784916e36f, low = a < 7.52316384526264e-37f;   // 2^120, 2^-120
    if (high || low) {
      a = high ? fminf(x, y) : fmaxf(x, y);
      b = high ? fmaxf(x, y) : fminf(x, y);
    }
  }
  __device__ __forceinline__ float operator()(float v, float bias) const { return fmaf(__fmul_rn(v, a), b, bias); }
};

// Stores alpha * v + bias for `jn` tokens from m on, of output feature n (one
// per lane: the lanes of a warp store neighbours).
template <int R>
__device__ __forceinline__ void store_tokens(const GemmArgs& a, int64_t m, int64_t n, int jn, const float* v, const Alpha& alpha,
                                             float bias) {
  const int64_t at = m * a.out_stride + n, step = a.out_stride;
  if (a.out_dtype == TS_F32) {
    float* p = reinterpret_cast<float*>(a.out) + at;
#pragma unroll
    for (int j = 0; j < R; ++j, p += step)
      if (j < jn) *p = alpha(v[j], bias);
  } else if (a.out_dtype == TS_BF16) {
    __nv_bfloat16* p = reinterpret_cast<__nv_bfloat16*>(a.out) + at;
#pragma unroll
    for (int j = 0; j < R; ++j, p += step)
      if (j < jn) *p = __float2bfloat16_rn(alpha(v[j], bias));
  } else {
    __half* p = reinterpret_cast<__half*>(a.out) + at;
#pragma unroll
    for (int j = 0; j < R; ++j, p += step)
      if (j < jn) *p = __float2half_rn(alpha(v[j], bias));
  }
}

__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// Stores alpha * v + bias as output features n .. n + 3 of token m.
__device__ __forceinline__ void store_four(const GemmArgs& a, int64_t m, int64_t n, const float4& v, const Alpha& alpha) {
  float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = alpha(f[i], a.bias && n + i < a.N ? load_f(a.bias, a.bias_dtype, n + i) : 0.f);
  const int64_t at = m * a.out_stride + n;
  if (a.out_dtype == TS_F32) {
    float* p = reinterpret_cast<float*>(a.out) + at;
    if (a.out_vec && n + 3 < a.N) {
      *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) p[i] = f[i];
    return;
  }
  uint16_t* p = reinterpret_cast<uint16_t*>(a.out) + at;
  uint2 w;
  if (a.out_dtype == TS_BF16) {
    w = make_uint2(paged::pack2<true>(f[0], f[1]), paged::pack2<true>(f[2], f[3]));
  } else {
    w = make_uint2(paged::pack2<false>(f[0], f[1]), paged::pack2<false>(f[2], f[3]));
  }
  if (a.out_vec && n + 3 < a.N) {
    *reinterpret_cast<uint2*>(p) = w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < a.N) p[i] = (uint16_t)((i < 2 ? w.x : w.y) >> (16 * (i & 1)));
}

// Work items of a CTA: a tile and the stages [k0, k1) of it that are its own.
struct Item {
  int tile, k0, k1;
};
struct ItemIter {
  int64_t u, u1;
};
__device__ __forceinline__ ItemIter items_begin(const GemmArgs& a, int ntiles) {
  const int64_t U = (int64_t)ntiles * a.kblocks;
  return {U * blockIdx.x / gridDim.x, U * (blockIdx.x + 1) / gridDim.x};
}
__device__ __forceinline__ bool items_next(const GemmArgs& a, ItemIter& it, Item& x) {
  if (it.u >= it.u1) return false;
  x.tile = (int)(it.u / a.kblocks);
  x.k0 = (int)(it.u - (int64_t)x.tile * a.kblocks);
  x.k1 = (int)min((int64_t)a.kblocks, x.k0 + (it.u1 - it.u));
  it.u += x.k1 - x.k0;
  return true;
}

// A lane's 16 columns of a row of tokens from p on, of which `left` exist.
template <int DT>
__device__ __forceinline__ void load_run(const typename Elem<DT>::T* p, int left, bool aligned, Lane<DT>& v) {
  constexpr int N = Lane<DT>::N;
  if (aligned && left >= 16) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + i);
      v.w[4 * i] = u.x; v.w[4 * i + 1] = u.y; v.w[4 * i + 2] = u.z; v.w[4 * i + 3] = u.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v.w[i] = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < left) {
      if (DT == TS_F32) v.w[i % N] = (uint32_t)p[i];
      else v.w[(i / 2) % N] |= (uint32_t)p[i] << (16 * (i & 1));
    }
}

// Quantises columns [256 kb, 256 kb + 256) of all tokens into a stage: codes as
// TMA would swizzle them, scales as a scale tile lays them. The loads are on
// their way while the warp waits for the stage (`ready`). By a whole warp, 16
// lanes a row.
template <bool NV, int DT, typename Ready>
__device__ __forceinline__ bool quantise_stage(const GemmArgs& a, int kb, char* sx, char* ssx, float g, float to_scale,
                                               Ready ready) {
  using T = typename Elem<DT>::T;
  constexpr int kAhead = 4;                        // rows of a lane in flight
  const int lane = threadIdx.x & 31, j = lane & 15, M = (int)a.M;
  const int64_t c0 = (int64_t)kb * kBK + j * 16;
  const int left = (int)max((int64_t)0, min((int64_t)16, a.K - c0));
  const int block = NV ? j : j >> 1;               // of the stage
  for (int r0 = 0; r0 < M; r0 += 2 * kAhead) {
    Lane<DT> v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int r = r0 + 2 * k + (lane >> 4);
      load_run<DT>(reinterpret_cast<const T*>(a.x) + (r < M ? r * a.x_stride + c0 : 0), r < M ? left : 0, a.x_aligned, v[k]);
    }
    if (r0 == 0 && !ready()) return false;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (r0 + 2 * k >= M) break;
      const int r = r0 + 2 * k + (lane >> 4);
      uint2 codes;
      const uint32_t sc = quantise16<DT, NV>(v[k], g, to_scale, codes);
      if (r >= M) continue;
      *reinterpret_cast<uint2*>(sx + r * 128 + (((j >> 1) ^ (r & 7)) << 4) + (j & 1) * 8) = codes;
      if (NV || (j & 1) == 0) ssx[(block >> 2) * kTileBytes + r * 16 + (block & 3)] = (char)sc;
    }
  }
  return true;
}

template <bool NV, int BT, bool Q>
__global__ void __launch_bounds__(kThreads + (Q ? kQuantWarps * 32 : 0), 1) fp4_gemm_kernel(const __grid_constant__ CUtensorMap wmap,
                                                            const __grid_constant__ CUtensorMap xmap,
                                                            const GemmArgs a) {
  using P = Shape<NV, BT>;
  static_assert(!Q || BT <= 32, "the tokens' scales lie in a tile's first 32 rows");
  constexpr int S = P::S;
  extern __shared__ char smem_raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  char* s_w = smem;                                  // [S][128][128]
  char* s_x = s_w + S * kABytes;                     // [S][BT][128]
  char* s_sw = s_x + S * P::kXBytes;                 // [S][tiles][512]
  char* s_sx = s_sw + S * P::kSf;                    // the same of the tokens
  uint64_t* full = reinterpret_cast<uint64_t*>(s_sx + S * P::kSf);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + P::kAcc;
  uint64_t* drain = tempty + P::kAcc;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  int* epi_flag = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ntiles = a.wblocks * a.tblocks;
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&wmap);
    if (!Q) prefetch_tensormap(&xmap);
    for (int i = 0; i < S; ++i) {
      mbar_init(full + i, Q ? 2 : 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < P::kAcc; ++i) {
      mbar_init(tfull + i, 1);
      mbar_init(tempty + i, kEpiWarps * 32);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      auto load_w = [&](const Item& x, int kb, int s) {
        const int wb = x.tile / a.tblocks, t0 = kb * P::kTiles;
        const uint32_t sf_bytes = min(P::kTiles, a.kt - t0) * kTileBytes;
        mbar_arrive_expect_tx(full + s, Q ? kABytes + sf_bytes : kABytes + P::kXBytes + 2 * sf_bytes);
        tma_load_2d(s_w + s * kABytes, &wmap, kb * 128, wb * kBW, full + s);
        bulk_load(s_sw + s * P::kSf, a.wscales + ((int64_t)wb * a.kt + t0) * kTileBytes, sf_bytes, full + s);
      };
      auto load_x = [&](const Item& x, int kb, int s) {
        const int tb = x.tile % a.tblocks, t0 = kb * P::kTiles;
        const uint32_t sf_bytes = min(P::kTiles, a.kt - t0) * kTileBytes;
        tma_load_2d(s_x + s * P::kXBytes, &xmap, kb * 128, tb * BT, full + s);
        // (tb > 0 only with BT = 128: token tiles are scale tiles)
        bulk_load(s_sx + s * P::kSf, a.xscales + ((int64_t)tb * a.kt + t0) * kTileBytes, sf_bytes, full + s);
      };
      // The weight's first S stages are loaded while the kernel that writes
      // the tokens' codes may still run; everything else follows its end.
      const int ahead = a.stall ? 0 : (int)min((int64_t)S, items_begin(a, ntiles).u1 - items_begin(a, ntiles).u);
      int s = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = !a.stall;
      Item x;
      ItemIter it = items_begin(a, ntiles);
      while (issued < ahead && items_next(a, it, x))
        for (int kb = x.k0; kb < x.k1 && issued < ahead; ++kb) load_w(x, kb, issued++);
      pdl_wait_primary();
      issued = 0;
      it = items_begin(a, ntiles);
      while (ok && items_next(a, it, x)) {
        for (int kb = x.k0; kb < x.k1; ++kb) {
          if (issued >= ahead) {
            if (!mbar_wait_hint(empty + s, ph ^ 1, &g_err, 21, a.wait_ns)) {
              ok = false;
              break;
            }
            load_w(x, kb, s);
          }
          if (!Q) load_x(x, kb, s);
          ++issued;
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      // the CTA's own copies have landed before it ends (after another
      // role's timeout nobody else waits for them)
      for (int i = 0; i < S && i < issued; ++i) {
        s = s == 0 ? S - 1 : s - 1;
        if (s == S - 1) ph ^= 1;
        mbar_wait_hint(full + s, ph, nullptr, 0, a.wait_ns);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint64_t wd0 = umma_desc_sw128(smem_u32(s_w)), xd0 = umma_desc_sw128(smem_u32(s_x));
      const uint64_t swd0 = desc_scales(smem_u32(s_sw)), sxd0 = desc_scales(smem_u32(s_sx));
      const uint32_t sf0 = tmem + P::kAcc * P::kAccCols;
      int s = 0, buf = 0;
      uint32_t ph = 0, bph = 0;
      ItemIter it = items_begin(a, ntiles);
      Item x;
      bool ok = true;
      while (ok && items_next(a, it, x)) {
        if (!mbar_wait_hint(tempty + buf, bph ^ 1, &g_err, 22, a.wait_ns)) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * P::kAccCols;
        for (int kb = x.k0; kb < x.k1; ++kb) {
          if (!mbar_wait_hint(full + s, ph, &g_err, 23, a.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sfa = sf0 + s * P::kSfCols, sfb = sfa + 4 * P::kTiles;
          const int nt = min(P::kTiles, a.kt - kb * P::kTiles);
          for (int t = 0; t < nt; ++t) {
            const uint64_t at = (uint64_t)((s * P::kSf + t * kTileBytes) >> 4);
            copy_scales(sfa + 4 * t, swd0 + at);
            copy_scales(sfb + 4 * t, sxd0 + at);
          }
          const int nk = min(kBK / kColPad, a.steps - kb * (kBK / kColPad));
          const uint64_t wd = wd0 + (uint64_t)((s * kABytes) >> 4), xd = xd0 + (uint64_t)((s * P::kXBytes) >> 4);
          for (int k = 0; k < nk; ++k) {
            const int t = NV ? k : k >> 1;
            const uint32_t sf = NV ? 0u : (uint32_t)(k & 1) * 2;
            mma_fp4<NV>(d, wd + 2 * k, xd + 2 * k, idesc_fp4<NV>(kBW, BT, sf), sfa + 4 * t,
                        sfb + 4 * t, (kb != x.k0 || k != 0) ? 1u : 0u);
          }
          umma_commit(empty + s);
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
        }
        if (ok) umma_commit(tfull + buf);
        if (++buf == P::kAcc) {
          buf = 0;
          bph ^= 1;
        }
      }
      // every MMA issued has finished before the TMEM is freed
      umma_commit(drain);
      mbar_wait_hint(drain, 0, nullptr, 0, a.wait_ns);
    }
  } else if (Q && warp >= 2 + kEpiWarps) {
    const float g = usable_scale(a.xg), to_scale = NV ? __frcp_rn(__fmul_rn(6.f, g)) : 0.f;
    int n = 0;                                         // of the CTA's stages
    bool ok = true;
    ItemIter it = items_begin(a, ntiles);
    Item x;
    while (ok && items_next(a, it, x)) {
      for (int kb = x.k0; kb < x.k1; ++kb, ++n) {
        if (n % kQuantWarps != warp - (2 + kEpiWarps)) continue;
        const int s = n % S;
        auto ready = [&] {
          return __all_sync(0xffffffffu, mbar_wait_hint(empty + s, (uint32_t)(n / S & 1) ^ 1, &g_err, 25, a.wait_ns));
        };
        char* sx = s_x + s * P::kXBytes;
        char* ssx = s_sx + s * P::kSf;
        if (a.x_dtype == TS_BF16) ok = quantise_stage<NV, TS_BF16>(a, kb, sx, ssx, g, to_scale, ready);
        else if (a.x_dtype == TS_F16) ok = quantise_stage<NV, TS_F16>(a, kb, sx, ssx, g, to_scale, ready);
        else ok = quantise_stage<NV, TS_F32>(a, kb, sx, ssx, g, to_scale, ready);
        if (!ok) break;
        fence_proxy_async_smem();                      // the tensor cores read what was written
        __syncwarp();
        if (lane == 0) mbar_arrive(full + s);
      }
    }
  } else {
    const int quad = warp & 3;
    const int r = quad * 32 + lane;                  // this thread's row of the tile
    const Alpha alpha(usable_scale(a.wg), usable_scale(a.xg));
    constexpr int CW = BT < 32 ? 16 : 32;
    int buf = 0;
    uint32_t bph = 0;
    ItemIter it = items_begin(a, ntiles);
    Item x;
    while (items_next(a, it, x)) {
      const int64_t m0 = (int64_t)(x.tile % a.tblocks) * BT;
      const int64_t n = (int64_t)(x.tile / a.tblocks) * kBW + r;
      if (!named_bar_and(3, kEpiWarps * 32, mbar_wait_hint(tfull + buf, bph, &g_err, 24, a.wait_ns))) break;
      tc_fence_after();
      const bool valid = n < a.N;
      const bool whole = x.k0 == 0 && x.k1 == a.kblocks;
      const int jn_all = (int)min((int64_t)BT, a.M - m0);
      float* pp = whole ? nullptr : a.partials + ((size_t)blockIdx.x * 2 + (x.k0 > 0 ? 0 : 1)) * (BT * kBW);
      const float bias = a.bias && valid ? load_f(a.bias, a.bias_dtype, n) : 0.f;
      const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + buf * P::kAccCols;
      if (a.cluster) {
        // to shared memory, over the stages (all used): [BT tokens][128 rows]
        // (the CTA's only item: nobody waits for the accumulator)
#pragma unroll 1
        for (int c = 0; c < BT / CW && c * CW < jn_all; ++c) {
          float v[CW];
          if constexpr (CW == 32) tmem_ld32(acc + c * CW, v);
          else tmem_ld16(acc + c * CW, v);
          float* dst = reinterpret_cast<float*>(s_w) + c * CW * kBW + r;
#pragma unroll
          for (int j = 0; j < CW; ++j) dst[j * kBW] = v[j];
        }
        break;
      }
#pragma unroll 1
      for (int c = 0; c < BT / CW; ++c) {
        float v[CW];
        if constexpr (CW == 32) tmem_ld32(acc + c * CW, v);
        else tmem_ld16(acc + c * CW, v);
        if (c == BT / CW - 1) {
          tc_fence_before();
          mbar_arrive(tempty + buf);
        }
        if (!whole) {
          // a piece: [BT / 4 tokens][128 rows][4 tokens], coalesced both ways
          float4* dst = reinterpret_cast<float4*>(pp) + (size_t)(c * CW / 4) * kBW + r;
#pragma unroll
          for (int j = 0; j < CW / 4; ++j)
            if (c * CW + 4 * j < jn_all) dst[j * kBW] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          continue;
        }
        if (!valid) continue;
        store_tokens<CW>(a, m0 + c * CW, n, min(CW, jn_all - c * CW), v, alpha, bias);
      }
      if (++buf == P::kAcc) {
        buf = 0;
        bph ^= 1;
      }
      if (whole) continue;
      // a tile split over several CTAs: the last to arrive adds the pieces
      named_bar_sync(3, kEpiWarps * 32);
      if (r == 0) {
        __threadfence();                               // the CTA's piece, before its arrival
        *epi_flag = atomicAdd(a.counters + x.tile, 1);
        __threadfence();
      }
      named_bar_sync(3, kEpiWarps * 32);
      const int64_t U = (int64_t)ntiles * a.kblocks;
      const int G = gridDim.x;
      const int64_t u_lo = (int64_t)x.tile * a.kblocks, u_hi = u_lo + a.kblocks - 1;
      const int c_first = (int)(((u_lo + 1) * G - 1) / U), c_last = (int)(((u_hi + 1) * G - 1) / U);
      const int old = *epi_flag;
      named_bar_sync(3, kEpiWarps * 32);
      if (old != c_last - c_first) continue;
      if (r == 0) a.counters[x.tile] = 0;
      if (!valid) continue;
      // the tile's beginning lies in its CTA's second slot, the other pieces
      // in their CTAs' first; kRun tokens of 4 pieces in flight
      constexpr int kPiece4 = BT * kBW / 4;
      const float4* base = reinterpret_cast<const float4*>(a.partials) + (size_t)c_first * 2 * kPiece4 + r;
      const int pieces = c_last - c_first + 1;
      constexpr int kRun = BT < 32 ? BT : 32, kRun4 = kRun / 4;   // tokens of a round
      for (int j0 = 0; j0 < jn_all; j0 += kRun) {
        float4 sum[kRun4];
#pragma unroll
        for (int u = 0; u < kRun4; ++u) sum[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < pieces; c += 4) {
          // (tokens behind the last one were not written: read, never stored)
          float4 t[4][kRun4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int cc = min(c + i, pieces - 1);
            const float4* src = base + (cc == 0 ? (size_t)kPiece4 : (size_t)cc * 2 * kPiece4) + (size_t)(j0 / 4) * kBW;
#pragma unroll
            for (int u = 0; u < kRun4; ++u) t[i][u] = __ldcg(src + u * kBW);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (c + i >= pieces) break;
#pragma unroll
            for (int u = 0; u < kRun4; ++u) {
              sum[u].x += t[i][u].x;
              sum[u].y += t[i][u].y;
              sum[u].z += t[i][u].z;
              sum[u].w += t[i][u].w;
            }
          }
        }
        float f[kRun];
#pragma unroll
        for (int u = 0; u < kRun4; ++u) {
          f[4 * u] = sum[u].x;
          f[4 * u + 1] = sum[u].y;
          f[4 * u + 2] = sum[u].z;
          f[4 * u + 3] = sum[u].w;
        }
        store_tokens<kRun>(a, m0 + j0, n, min(kRun, jn_all - j0), f, alpha, bias);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
  if (a.cluster) {
    // every CTA of the tile has its sums in shared memory: a warp adds a
    // token's, four neighbouring features per lane
    static_assert((size_t)BT * kBW * 4 <= (size_t)S * kABytes, "the sums lie over the stages");
    constexpr int kWarpsAll = kThreads / 32 + (Q ? kQuantWarps : 0);
    cluster_sync();
    const int rank = (int)cta_rank(), tile = blockIdx.x / a.cluster;
    const int64_t m0 = (int64_t)(tile % a.tblocks) * BT, n = (int64_t)(tile / a.tblocks) * kBW + 4 * lane;
    const int jn = (int)min((int64_t)BT, a.M - m0);
    const Alpha alpha(usable_scale(a.wg), usable_scale(a.xg));
    for (int j = rank + a.cluster * warp; j < jn; j += a.cluster * kWarpsAll) {
      const uint32_t at = smem_u32(s_w) + (uint32_t)(j * kBW + 4 * lane) * 4;
      float4 v[kMaxCluster];
#pragma unroll
      for (int p = 0; p < kMaxCluster; ++p)
        if (p < a.cluster) v[p] = ld_cluster(map_cta(at, p));
#pragma unroll
      for (int p = 1; p < kMaxCluster; ++p)
        if (p < a.cluster) {
          v[0].x += v[p].x;
          v[0].y += v[p].y;
          v[0].z += v[p].z;
          v[0].w += v[p].w;
        }
      if (n < a.N) store_four(a, m0 + j, n, v[0], alpha);
    }
    cluster_sync();                                    // nobody leaves while its sums may be read
  }
}

// ---- prefill: tiles of 256 tokens x 256 weight rows on CTA pairs ------------------
//
// Two CTAs of a cluster share one MMA (cta_group::2, M = 256): each holds its
// 128 token rows of A, half of B's rows and the accumulator of its own
// tokens, so every operand byte is fetched by one of the two and feeds both
// tensor cores; a stage of 256 columns brings 38 KB per CTA for 128 x BN x 256
// products where a lone CTA's 128 x 256 tile needs 54 KB. Loads of both CTAs
// complete on the leader's barrier; the leader's thread issues scale copies
// and MMAs for both; commits release the stage in both. Tokens are the
// accumulator's lanes, so that a thread stores runs of its token's outputs.
// Measured: 8192 x 28672 x 8192 nvfp4, 720 to 815 us by card and by what ran
// before, 4.7 to 5.3 PFLOP/s at the power limit (a lone CTA's tiles of 128 x 128:
// 1284 us); 2047 x 14336 x 4096, 62 us, 3.9 PFLOP/s, in seven rounds of tiles where six hold all but four.
// Bound by the loads into each SM (about 52 of 64 bytes a clock).

constexpr int BN = 256, kHalf = BN / 2;
constexpr int kPairEpi = 8, kPairThreads = (2 + kPairEpi) * 32;
constexpr int kOutWords = 32 * 17;         // an epilogue warp's staging: 32 rows of 16 words, one word apart

template <bool NV>
struct Pair {
  static constexpr int kTiles = NV ? 4 : 2;                    // scale tiles of a stage, per 128 rows
  static constexpr int kRowTiles = BN / 128;
  static constexpr int kBBytes = BN / 2 * 128;
  static constexpr int kSfA = kTiles * kTileBytes;
  static constexpr int kSfB = kRowTiles * kSfA;
  static constexpr int kStage = kABytes + kBBytes + kSfA + kSfB;
  static constexpr int kSfCols = 4 * kTiles * (1 + kRowTiles);
  static constexpr int kFitTmem = (kTmemCols - BN) / kSfCols;
  static constexpr int kEpi = 128 + kPairEpi * (kHalf + kOutWords) * 4;   // barriers, then the epilogue warps' words
  static constexpr int kFitSmem = (227 * 1024 - 1024 - kEpi) / kStage;
  static constexpr int S = kFitTmem < kFitSmem ? kFitTmem : kFitSmem;
  static_assert((2 * S + 3) * 8 + 4 <= 128, "barriers");
  static constexpr size_t kSmem = 1024 + (size_t)S * kStage + kEpi;
};

struct PairArgs {
  const float* wg;
  const float* xg;
  int64_t M, N;
  int mblocks, nblocks, kblocks;
  int kt, steps;
  const void* bias;
  int bias_dtype;
  void* out;
  int out_dtype;
  int64_t out_stride;
  int vec;                         // rows of out take 16-byte stores
  uint64_t wait_ns;
  int stall, overlap;
};

// 128 consecutive fp32 columns of this warp's TMEM lane quadrant, four loads in flight.
__device__ __forceinline__ void tmem_ld128(uint32_t taddr, uint32_t (&r)[128]) {
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    uint32_t* q = r + 32 * h;
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]), "=r"(q[4]), "=r"(q[5]), "=r"(q[6]), "=r"(q[7]),
          "=r"(q[8]), "=r"(q[9]), "=r"(q[10]), "=r"(q[11]), "=r"(q[12]), "=r"(q[13]), "=r"(q[14]),
          "=r"(q[15]), "=r"(q[16]), "=r"(q[17]), "=r"(q[18]), "=r"(q[19]), "=r"(q[20]), "=r"(q[21]),
          "=r"(q[22]), "=r"(q[23]), "=r"(q[24]), "=r"(q[25]), "=r"(q[26]), "=r"(q[27]), "=r"(q[28]),
          "=r"(q[29]), "=r"(q[30]), "=r"(q[31])
        : "r"(taddr + 32 * h));
  }
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  // the registers hold the values from here on: no use moves before the wait
#pragma unroll
  for (int i = 0; i < 128; ++i) asm volatile("" : "+r"(r[i]));
}

// TMA tile load into this CTA's shared memory, completing on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void copy_scales_pair(uint32_t tmem, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
template <bool NV>
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
  if (NV)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

template <bool NV>
__global__ void __launch_bounds__(kPairThreads) __cluster_dims__(2, 1, 1)
    fp4_pair_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                    const __grid_constant__ CUtensorMap asmap, const __grid_constant__ CUtensorMap bsmap,
                    const PairArgs a) {
  using P = Pair<NV>;
  constexpr int S = P::S;
  extern __shared__ char smem_raw[];
  // both CTAs have one layout: the dynamic area starts at the same address in each
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  char* s_a = smem;
  char* s_b = s_a + S * kABytes;
  char* s_sa = s_b + S * P::kBBytes;
  char* s_sb = s_sa + S * P::kSfA;
  uint64_t* full = reinterpret_cast<uint64_t*>(s_sb + S * P::kSfB);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + 1;
  uint64_t* drain = tempty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  char* s_epi = reinterpret_cast<char*>(full) + 128;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int ntiles = a.mblocks * a.nblocks;
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&amap);
    prefetch_tensormap(&bmap);
    prefetch_tensormap(&asmap);
    prefetch_tensormap(&bsmap);
    for (int i = 0; i < S; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    mbar_init(tfull, 1);
    mbar_init(tempty, 2 * kPairEpi);
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    const bool leads = elect_one();
    if (leads) pdl_wait_primary();                     // (the kernel that writes the tokens' codes)
    if (leads && !a.stall) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < ntiles; tile += pairs) {
        const int mb = tile % a.mblocks, nb = tile / a.mblocks;
        const int arow = mb * 256 + (int)rank * 128, brow = nb * BN + (int)rank * (BN / 2);
        const int at = (mb * 2 + (int)rank) * a.kt, bt = nb * P::kRowTiles * a.kt;
        for (int kb = 0; kb < a.kblocks; ++kb) {
          if (!mbar_wait_hint(empty + s, ph ^ 1, &g_err, 31, a.wait_ns)) {
            ok = false;
            break;
          }
          // both CTAs' copies count on the leader's barrier
          const uint32_t bar = map_cta(smem_u32(full + s), 0);
          if (rank == 0) mbar_arrive_expect_tx(full + s, 2 * P::kStage);
          tma_load_pair(smem_u32(s_a + s * kABytes), &amap, kb * 128, arow, bar);
          tma_load_pair(smem_u32(s_b + s * P::kBBytes), &bmap, kb * 128, brow, bar);
          // scale tiles are rows of 512 bytes; tiles behind a row's end are
          // loaded too (of the next row, or zeros) and not used
          tma_load_pair(smem_u32(s_sa + s * P::kSfA), &asmap, 0, at + kb * P::kTiles, bar);
#pragma unroll
          for (int r = 0; r < P::kRowTiles; ++r)
            tma_load_pair(smem_u32(s_sb + s * P::kSfB + r * P::kSfA), &bsmap, 0, bt + r * a.kt + kb * P::kTiles, bar);
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      // every stage has been released to this CTA before it ends; after a
      // timeout, the copies in flight have landed
      for (int i = 0; i < S; ++i) {
        if (ok) {
          if (!mbar_wait_hint(empty + s, ph ^ 1, &g_err, 35, a.wait_ns)) break;
        } else if (rank == 0) {
          mbar_wait_hint(full + s, ph ^ 1, nullptr, 0, a.wait_ns);
        }
        if (++s == S) {
          s = 0;
          ph ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (rank != 0) {
      // the last commit reaches this CTA's barrier too: it stays until then
      if (elect_one()) mbar_wait_hint(drain, 0, nullptr, 0, a.wait_ns);
    } else if (elect_one()) {
      const uint64_t ad0 = umma_desc_sw128(smem_u32(s_a)), bd0 = umma_desc_sw128(smem_u32(s_b));
      const uint64_t sad0 = desc_scales(smem_u32(s_sa)), sbd0 = desc_scales(smem_u32(s_sb));
      const uint32_t sf0 = tmem + BN;
      int s = 0, n = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < ntiles; tile += pairs, ++n) {
        if (!mbar_wait_hint(tempty, (n & 1) ^ 1, &g_err, 32, a.wait_ns)) break;
        tc_fence_after();
        for (int kb = 0; kb < a.kblocks; ++kb) {
          if (!mbar_wait_hint(full + s, ph, &g_err, 33, a.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sfa = sf0 + s * P::kSfCols, sfb = sfa + 4 * P::kTiles;
#pragma unroll
          for (int t = 0; t < P::kTiles; ++t) {
            copy_scales_pair(sfa + 4 * t, sad0 + (uint64_t)((s * P::kSfA + t * kTileBytes) >> 4));
#pragma unroll
            for (int r = 0; r < P::kRowTiles; ++r)
              copy_scales_pair(sfb + 4 * (t * P::kRowTiles + r),
                               sbd0 + (uint64_t)((s * P::kSfB + r * P::kSfA + t * kTileBytes) >> 4));
          }
          const int nk = min(kBK / kColPad, a.steps - kb * (kBK / kColPad));
          const uint64_t ad = ad0 + (uint64_t)((s * kABytes) >> 4), bd = bd0 + (uint64_t)((s * P::kBBytes) >> 4);
#pragma unroll
          for (int k = 0; k < kBK / kColPad; ++k) {
            if (k < nk) {
              const int t = NV ? k : k >> 1;
              const uint32_t sf = NV ? 0u : (uint32_t)(k & 1) * 2;
              mma_pair<NV>(tmem, ad + 2 * k, bd + 2 * k, idesc_fp4<NV>(256, BN, sf), sfa + 4 * t,
                           sfb + 4 * t * P::kRowTiles, (kb != 0 || k != 0) ? 1u : 0u);
            }
          }
          commit_pair(empty + s);
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
        }
        if (ok) commit_pair(tfull);
      }
      // every MMA issued has finished before the TMEM is freed
      commit_pair(drain);
      mbar_wait_hint(drain, 0, nullptr, 0, a.wait_ns);
    }
  } else {
    // two warps per quadrant of TMEM lanes, each with half of the columns
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const Alpha alpha(usable_scale(a.wg), usable_scale(a.xg));
    const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + half * kHalf;
    const uint32_t free_bar = map_cta(smem_u32(tempty), 0);
    int n = 0;
    float* s_bias = reinterpret_cast<float*>(s_epi) + (warp - 2) * (kHalf + kOutWords);   // [128]
    uint32_t* s_out = reinterpret_cast<uint32_t*>(s_bias + kHalf);                         // [32 rows][17 words]
    for (int tile = pair; tile < ntiles; tile += pairs, ++n) {
      const int64_t m0 = (int64_t)(tile % a.mblocks) * 256 + rank * 128 + quad * 32;
      const int64_t n0 = (int64_t)(tile / a.mblocks) * BN + half * kHalf;
      const int cols = (int)max((int64_t)0, min((int64_t)kHalf, a.N - n0));
      const int rows = (int)max((int64_t)0, min((int64_t)32, a.M - m0));
      __syncwarp();                                    // (the last tile's biases have been used)
#pragma unroll
      for (int i = 0; i < kHalf / 32; ++i) {
        const int col = i * 32 + lane;
        s_bias[col] = a.bias != nullptr && col < cols ? load_f(a.bias, a.bias_dtype, n0 + col) : 0.f;
      }
      __syncwarp();
      const bool got = mbar_wait_hint(tfull, n & 1, &g_err, 34, a.wait_ns);
      if (!__all_sync(0xffffffffu, got)) break;
      tc_fence_after();
      // the sums wait in registers, so that the accumulator is free again
      // before the first of them is stored
      uint32_t v[kHalf];
      tmem_ld128(acc, v);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(free_bar);
      if (rows == 0) continue;
#pragma unroll
      for (int i = 0; i < kHalf; i += 4) {
        const float4 bs = *reinterpret_cast<const float4*>(s_bias + i);
        v[i] = __float_as_uint(alpha(__uint_as_float(v[i]), bs.x));
        v[i + 1] = __float_as_uint(alpha(__uint_as_float(v[i + 1]), bs.y));
        v[i + 2] = __float_as_uint(alpha(__uint_as_float(v[i + 2]), bs.z));
        v[i + 3] = __float_as_uint(alpha(__uint_as_float(v[i + 3]), bs.w));
      }
      if (a.out_dtype == TS_F32) {
        float* out = reinterpret_cast<float*>(a.out) + m0 * a.out_stride + n0;
        if (a.vec) {                                   // N is a multiple of 4
          float* row = out + lane * a.out_stride;
#pragma unroll
          for (int i = 0; i < kHalf; i += 4)
            if (lane < rows && i < cols) *reinterpret_cast<uint4*>(row + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          continue;
        }
        // 16 columns of the warp's rows at a time through shared memory, two
        // rows of them per store
#pragma unroll
        for (int c = 0; c < kHalf; c += 16) {
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 16; ++j) s_out[lane * 17 + j] = v[c + j];
          __syncwarp();
          const int col = c + (lane & 15);
          for (int r = lane >> 4; r < rows; r += 2)
            if (col < cols) out[r * a.out_stride + col] = __uint_as_float(s_out[r * 17 + (lane & 15)]);
        }
        continue;
      }
#pragma unroll
      for (int i = 0; i < kHalf / 2; ++i) {
        const float x = __uint_as_float(v[2 * i]), y = __uint_as_float(v[2 * i + 1]);
        if (a.out_dtype == TS_BF16) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
          v[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __half2 h = __floats2half2_rn(x, y);
          v[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + m0 * a.out_stride + n0;
      if (a.vec) {                                     // N is a multiple of 8
        uint16_t* row = out + lane * a.out_stride;
#pragma unroll
        for (int i = 0; i < kHalf / 8; ++i)
          if (lane < rows && i * 8 < cols)
            *reinterpret_cast<uint4*>(row + i * 8) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        continue;
      }
      // 32 columns of the warp's rows at a time through shared memory: two rows
      // per store where rows start on words, one row of elements otherwise
      const bool words = (reinterpret_cast<uintptr_t>(a.out) & 3) == 0 && (a.out_stride & 1) == 0;
#pragma unroll
      for (int c = 0; c < kHalf / 2; c += 16) {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 16; ++j) s_out[lane * 17 + j] = v[c + j];
        __syncwarp();
        if (words) {
          const int col = 2 * (c + (lane & 15));
          for (int r = lane >> 4; r < rows; r += 2) {
            const uint32_t x = s_out[r * 17 + (lane & 15)];
            uint16_t* dst = out + r * a.out_stride + col;
            if (col + 1 < cols) *reinterpret_cast<uint32_t*>(dst) = x;
            else if (col < cols) *dst = (uint16_t)x;
          }
        } else {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(s_out);
          for (int r = 0; r < rows; ++r)
            if (2 * c + lane < cols) out[r * a.out_stride + 2 * c + lane] = h[r * 34 + lane];
        }
      }
    }
  }

  // neither CTA leaves, nor frees TMEM, while the other's copies, MMAs or
  // arrivals may still reach it
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// ---- host -------------------------------------------------------------------

struct Plan {
  bool pair;        // CTA pairs on tiles of 256 tokens x 256 weight rows
  int BT, tblocks, wblocks, kblocks, ntiles, grid;
  int cluster;      // CTAs that share a tile as a cluster, or 0
};

// Clusters of `size` CTAs, one per SM, that the device holds at once.
static int max_clusters(int size) {
  static thread_local int known[kMaxCluster + 1], known_dev = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    (void)cudaGetLastError();
    return 0;
  }
  if (dev != known_dev) {
    for (int i = 0; i <= kMaxCluster; ++i) known[i] = -1;
    known_dev = dev;
  }
  if (known[size] < 0) {
    auto k = fp4_gemm_kernel<true, 128, false>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(sm_count() / size * size));
    cfg.blockDim = dim3((unsigned)kThreads);
    cfg.dynamicSmemBytes = Shape<true, 128>::kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cfg.dynamicSmemBytes) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, k, &cfg) != cudaSuccess) {
      (void)cudaGetLastError();
      return 0;
    }
    known[size] = n;
  }
  return known[size];
}

// Cycles that a call takes at least, as measured: a stage of a pair's tile 620
// and the change from tile to tile 2000; a stage of a lone CTA's tile 550, or what
// its bytes take at DRAM's rate; a join of up to four pieces 3000 and 2500 per
// 32 tokens, of a cluster 1500 and 600. Only their order matters.
static Plan plan(int64_t M, int64_t N, int64_t K) {
  Plan p{};
  const int sms = std::max(2, sm_count()), pairs = sms / 2;
  p.kblocks = (int)((padded_cols(K) + kBK - 1) / kBK);
  p.BT = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  p.wblocks = (int)((N + kBW - 1) / kBW);
  p.tblocks = (int)((M + p.BT - 1) / p.BT);
  const int64_t ntiles = (int64_t)p.wblocks * p.tblocks, units = ntiles * p.kblocks;
  const int rounds = (int)(std::min<int64_t>(M, p.BT) + 31) / 32;
  const double stream = (double)units * (kABytes + 2048) / 3300;   // the weight's bytes, at DRAM's bytes per cycle
  auto cost = [&](int64_t grid, int pieces) {
    const double own = (double)((units + grid - 1) / grid) * 550;
    return std::max(own, stream) + (pieces > 1 ? 3000 + 2500.0 * rounds * ((pieces + 3) / 4) : 0) +
           (double)((ntiles + grid - 1) / grid) * rounds * 400;
  };
  // whole tiles, or whole parts of them, where the SMs hold them all at once;
  // else, or if that is better, equal shares of all stages
  const int64_t all = std::min<int64_t>(units, sms);
  p.grid = (int)all;
  double best = cost(all, (int)std::min<int64_t>(p.kblocks, all / std::max<int64_t>(1, ntiles) + 2));
  for (int parts = 1; parts <= p.kblocks && ntiles * parts <= sms; ++parts) {
    const bool fits = parts > 1 && parts <= kMaxCluster && max_clusters(parts) >= ntiles;
    const double c = fits ? cost(ntiles * parts, 1) + 1500 + 600.0 * rounds : cost(ntiles * parts, parts);
    if (c < best) {
      best = c;
      p.grid = (int)(ntiles * parts);
      p.cluster = fits ? parts : 0;
    }
  }
  p.ntiles = (int)std::min<int64_t>(ntiles, INT32_MAX);
  if (M <= 128) return p;
  const int64_t mb = (M + 255) / 256, nb = (N + BN - 1) / BN;
  const double pair = (double)((mb * nb + pairs - 1) / pairs) * (620.0 * p.kblocks + 2000);
  if (pair <= best || ntiles > (int64_t)paged::kCounters) {
    p.pair = true;
    p.cluster = 0;
    p.tblocks = (int)mb;
    p.wblocks = (int)nb;
    p.ntiles = (int)(mb * nb);
    p.grid = 2 * (int)std::min<int64_t>(mb * nb, pairs);
  }
  return p;
}

// Launch; with `overlap` the kernel may start while the one before it (which
// allows that, and whose results it waits for by itself) still runs.
template <typename K, typename... Args>
static cudaError_t launch_after(K k, int grid, int threads, size_t smem, cudaStream_t st, int overlap, int cluster,
                                const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (overlap) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  return cudaLaunchKernelEx(&cfg, k, args...);
}

template <bool NV>
static int launch_pair(const CUtensorMap (&m)[4], const PairArgs& a, int grid, cudaStream_t st) {
  auto k = fp4_pair_kernel<NV>;
  constexpr size_t smem = Pair<NV>::kSmem;
  static_assert(smem <= 227 * 1024, "shared memory");
  static thread_local int configured_dev = -1;
  int dev = 0;
  TS_CUDA_TRY(cudaGetDevice(&dev));
  if (configured_dev != dev) {
    TS_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    configured_dev = dev;
  }
  TS_CUDA_TRY(launch_after(k, grid, kPairThreads, smem, st, a.overlap, 0, m[0], m[1], m[2], m[3], a));
  TS_LAUNCH_CHECK();
  return TS_OK;
}

// Tensor map of a tensor's scale tiles: rows of 512 bytes, boxes of the tiles of a stage.
static int scale_map(CUtensorMap* map, const ts_fp4_tensor& t) {
  const uint64_t rows = (uint64_t)((t.rows + kTileRows - 1) / kTileRows) * scale_tiles(t.cols, t.format);
  return encode_tmap_2d(map, t.scales, CU_TENSOR_MAP_DATA_TYPE_UINT16, kTileBytes / 2, rows, kTileBytes, kTileBytes / 2,
                        kBK / block_of(t.format) / 4, CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <bool NV, int BT, bool Q>
static int launch(const CUtensorMap& wm, const CUtensorMap& xm, const GemmArgs& a, int grid, cudaStream_t st) {
  auto k = fp4_gemm_kernel<NV, BT, Q>;
  constexpr size_t smem = Shape<NV, BT>::kSmem;
  static_assert(smem <= 227 * 1024, "shared memory");
  static thread_local int configured_dev = -1;
  int dev = 0;
  TS_CUDA_TRY(cudaGetDevice(&dev));
  if (configured_dev != dev) {
    TS_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    configured_dev = dev;
  }
  TS_CUDA_TRY(launch_after(k, grid, kThreads + (Q ? kQuantWarps * 32 : 0), smem, st, a.overlap, a.cluster, wm, xm, a));
  TS_LAUNCH_CHECK();
  return TS_OK;
}

template <bool NV>
static int launch(int BT, const CUtensorMap& wm, const CUtensorMap& xm, const GemmArgs& a, int grid, cudaStream_t st) {
  static_assert(kOwnTokens <= 16, "tokens of the kernel that quantises them");
  if (a.x != nullptr) return launch<NV, 16, true>(wm, xm, a, grid, st);
  switch (BT) {
    case 16: return launch<NV, 16, false>(wm, xm, a, grid, st);
    case 32: return launch<NV, 32, false>(wm, xm, a, grid, st);
    case 64: return launch<NV, 64, false>(wm, xm, a, grid, st);
    default: return launch<NV, 128, false>(wm, xm, a, grid, st);
  }
}

}  // namespace fp4

}  // namespace ts

using namespace ts;
using namespace ts::fp4;

// Bytes of a plan's workspace: counters, then partial sums.
static size_t plan_bytes(const Plan& p) {
  return paged::kCounterBytes + (!p.pair && !p.cluster ? (size_t)p.grid * 2 * kBW * p.BT * 4 : 0);
}

extern "C" size_t ts_fp4_matmul_workspace_size(int64_t M, int64_t N, int64_t K, int format) {
  (void)format;
  if (M <= 0 || N <= 0 || K <= 0) return paged::kCounterBytes;
  return plan_bytes(plan(M, N, K));
}

// Tokens that the product quantises itself.
struct Tokens {
  const void* x;
  int dtype;
  int64_t stride;
};

static int matmul(const Plan& p, const ts_fp4_tensor* x, const ts_fp4_tensor* w, const void* bias, int bias_dtype, void* out,
                  int out_dtype, int64_t out_row_stride, void* workspace, size_t workspace_bytes, int overlap,
                  const Tokens* own, void* stream) {
  int rc;
  TS_UNSUPPORTED(out_dtype == TS_F16 || out_dtype == TS_BF16 || out_dtype == TS_F32, "unknown output type %d", out_dtype);
  TS_UNSUPPORTED(!bias || bias_dtype == TS_F16 || bias_dtype == TS_BF16 || bias_dtype == TS_F32, "unknown bias type %d",
                 bias_dtype);
  TS_REQUIRE(out, "NULL pointer");
  const size_t need = plan_bytes(p);
  if (!p.pair && (workspace == nullptr || workspace_bytes < need)) {
    set_error("workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return TS_ERR_WORKSPACE;
  }
  TS_REQUIRE(is_aligned(workspace, 16), "workspace must be 16-byte aligned");
  TS_UNSUPPORTED(p.pair || p.ntiles <= (int)paged::kCounters, "too many output features in one call");
  const float* wg = w->format == TS_NVFP4 ? w->global_scale : nullptr;
  const float* xg = x->format == TS_NVFP4 ? x->global_scale : nullptr;
  const int kt = (int)scale_tiles(w->cols, w->format), steps = (int)(padded_cols(w->cols) / kColPad);
  const uint64_t row = (uint64_t)padded_cols(w->cols) / 2;
  const int stall = take_test_stall() ? 1 : 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p.pair) {
    PairArgs a;
    a.wg = wg;
    a.xg = xg;
    a.M = x->rows;
    a.N = w->rows;
    a.mblocks = p.tblocks;
    a.nblocks = p.wblocks;
    a.kblocks = p.kblocks;
    a.kt = kt;
    a.steps = steps;
    a.bias = bias;
    a.bias_dtype = bias_dtype;
    a.out = out;
    a.out_dtype = out_dtype;
    a.out_stride = out_row_stride;
    const int per = out_dtype == TS_F32 ? 4 : 8;     // values of a 16-byte store
    a.vec = w->rows % per == 0 && out_row_stride % per == 0 && is_aligned(out, 16);
    a.wait_ns = wait_limit_ns();
    a.stall = stall;
    a.overlap = overlap;
    CUtensorMap m[4];
    rc = encode_tmap_2d(&m[0], x->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, row, (uint64_t)x->rows, row, 128, 128,
                        CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc == TS_OK)
      rc = encode_tmap_2d(&m[1], w->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, row, (uint64_t)w->rows, row, 128, BN / 2,
                          CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc == TS_OK) rc = scale_map(&m[2], *x);
    if (rc == TS_OK) rc = scale_map(&m[3], *w);
    if (rc != TS_OK) return rc;
    return w->format == TS_NVFP4 ? launch_pair<true>(m, a, p.grid, st) : launch_pair<false>(m, a, p.grid, st);
  }
  GemmArgs a;
  a.wscales = w->scales;
  a.xscales = x->scales;
  a.wg = wg;
  a.xg = xg;
  a.M = x->rows;
  a.N = w->rows;
  a.wblocks = p.wblocks;
  a.tblocks = p.tblocks;
  a.kblocks = p.kblocks;
  a.kt = kt;
  a.steps = steps;
  a.bias = bias;
  a.bias_dtype = bias_dtype;
  a.out = out;
  a.out_dtype = out_dtype;
  a.out_stride = out_row_stride;
  a.counters = reinterpret_cast<int*>(workspace);
  a.partials = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + paged::kCounterBytes);
  a.wait_ns = wait_limit_ns();
  a.stall = stall;
  a.overlap = overlap;
  a.x = own ? own->x : nullptr;
  a.x_dtype = own ? own->dtype : 0;
  a.x_stride = own ? own->stride : 0;
  a.x_aligned = own && is_aligned(own->x, 16) && own->stride * (own->dtype == TS_F32 ? 4 : 2) % 16 == 0;
  a.K = w->cols;
  a.cluster = p.cluster;
  const int wide = out_dtype == TS_F32 ? 16 : 8;       // bytes of four values
  a.out_vec = is_aligned(out, wide) && out_row_stride % 4 == 0;
  CUtensorMap wm, xm;
  rc = encode_tmap_2d(&wm, w->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, row, (uint64_t)w->rows, row, 128, kBW,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != TS_OK) return rc;
  if (own) xm = wm;                                    // (not used)
  else rc = encode_tmap_2d(&xm, x->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, row, (uint64_t)x->rows, row, 128, p.BT,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != TS_OK) return rc;
  return w->format == TS_NVFP4 ? launch<true>(p.BT, wm, xm, a, p.grid, st) : launch<false>(p.BT, wm, xm, a, p.grid, st);
}

extern "C" int ts_fp4_matmul(const ts_fp4_tensor* a, const ts_fp4_tensor* b, const void* bias, int bias_dtype, void* out,
                             int out_dtype, int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                             void* stream) {
  int rc = check_tensor(a, "ts_fp4_matmul a");
  if (rc != TS_OK) return rc;
  rc = check_tensor(b, "ts_fp4_matmul b");
  if (rc != TS_OK) return rc;
  TS_REQUIRE(a->format == b->format, "both operands must have one format");
  TS_REQUIRE(a->cols == b->cols, "a has %lld columns, b %lld", (long long)a->cols, (long long)b->cols);
  if (a->rows == 0 || b->rows == 0) return TS_OK;
  return matmul(plan(a->rows, b->rows, b->cols), a, b, bias, bias_dtype, out, out_dtype, out_row_stride, workspace,
                workspace_bytes, 0, nullptr, stream);
}

extern "C" size_t ts_serving_counter_bytes(void) { return paged::kCounterBytes; }

extern "C" int ts_fp4_status(void* workspace, size_t workspace_bytes, int clear, void* stream) {
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  TS_REQUIRE(workspace == nullptr || workspace_bytes >= paged::kCounterBytes, "workspace of %zu bytes, %zu needed",
             workspace_bytes, paged::kCounterBytes);
  int v = 0;
  TS_CUDA_TRY(cudaMemcpyFromSymbolAsync(&v, g_err, sizeof(int), 0, cudaMemcpyDeviceToHost, st));
  TS_CUDA_TRY(cudaStreamSynchronize(st));
  if (v == 0) return TS_OK;
  if (clear) {
    // the flag, and the counters that CTAs which gave up may have left
    const int zero = 0;
    TS_CUDA_TRY(cudaMemcpyToSymbolAsync(g_err, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st));
    if (workspace != nullptr) TS_CUDA_TRY(cudaMemsetAsync(workspace, 0, paged::kCounterBytes, st));
    TS_CUDA_TRY(cudaStreamSynchronize(st));
  }
  set_error("a bounded wait in the fp4 product ran out (code %d); the outputs of the calls since the last "
            "status check are not valid", v);
  return TS_ERR_TIMEOUT;
}

// ---- quantised activations and the product in one call ----------------------

static size_t linear_act_bytes(int64_t M, int64_t K, int format) {
  return align_up((size_t)M * (size_t)(padded_cols(K) / 2), 256) + align_up(ts_fp4_scales_bytes(M, K, format), 256);
}

extern "C" size_t ts_fp4_linear_workspace_size(int64_t M, int64_t N, int64_t K, int format) {
  if (M <= 0 || N <= 0 || K <= 0) return paged::kCounterBytes;
  return align_up(ts_fp4_matmul_workspace_size(M, N, K, format), 256) + linear_act_bytes(M, K, format);
}

extern "C" int ts_fp4_linear(const void* x, int x_dtype, int64_t M, int64_t x_row_stride, float* x_scale,
                             const ts_fp4_tensor* w, const void* bias, int bias_dtype, void* out, int out_dtype,
                             int64_t out_row_stride, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_tensor(w, "ts_fp4_linear w");
  if (rc != TS_OK) return rc;
  TS_REQUIRE(M >= 0, "bad shape");
  if (M == 0 || w->rows == 0) return TS_OK;
  const Plan p = plan(M, w->rows, w->cols);
  // the activations' codes and scales lie behind the product's scratch
  const size_t at = align_up(plan_bytes(p), 256), need = at + linear_act_bytes(M, w->cols, w->format);
  if (workspace == nullptr || workspace_bytes < need) {
    set_error("workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return TS_ERR_WORKSPACE;
  }
  TS_REQUIRE(is_aligned(workspace, 16), "workspace must be 16-byte aligned");
  ts_fp4_tensor t{};
  t.codes = reinterpret_cast<uint8_t*>(workspace) + at;
  t.scales = t.codes + align_up((size_t)M * (size_t)(padded_cols(w->cols) / 2), 256);
  t.global_scale = w->format == TS_NVFP4 ? x_scale : nullptr;
  t.rows = M;
  t.cols = w->cols;
  t.format = w->format;
  if (M <= kOwnTokens) {
    TS_UNSUPPORTED(x_dtype == TS_F16 || x_dtype == TS_BF16 || x_dtype == TS_F32, "unknown element type %d", x_dtype);
    TS_REQUIRE(x, "NULL pointer");
    const Tokens own = {x, x_dtype, x_row_stride};
    return matmul(p, &t, w, bias, bias_dtype, out, out_dtype, out_row_stride, workspace, at, 0, &own, stream);
  }
  rc = ts_fp4_quantize(x, x_dtype, x_row_stride, &t, 0, nullptr, 0, stream);
  if (rc != TS_OK) return rc;
  return matmul(p, &t, w, bias, bias_dtype, out, out_dtype, out_row_stride, workspace, at, 1, nullptr, stream);
}
