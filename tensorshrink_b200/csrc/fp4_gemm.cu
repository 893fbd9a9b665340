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
// A tile is 128 rows of b (the weight's output features; the MMA's M) x BT
// rows of a (tokens; its N), K in stages of 256. Roles in one persistent CTA
// per SM:
//   warp 0      TMA producer: codes of both operands (128-byte rows, 128-byte
//               swizzle) and, as bulk copies, the scale tiles of the stage
//   warp 1      one thread copies the stage's scale tiles to TMEM
//               (tcgen05.cp, broadcast to the four lane quadrants) and issues
//               the stage's MMAs. Scales have TMEM columns per stage: a
//               stage's columns are rewritten only after the MMAs that read
//               them have released the stage.
//   warps 2-5   epilogue: tcgen05.ld, tensor scales, bias, stores
//
// Decode-sized calls are bound by the weight's bytes, prefill by the tensor
// cores. Few tokens make few tiles: their stages are laid end to end and each
// CTA takes an equal share (split along K), partial sums being added by the
// last CTA of a tile to arrive, in CTA order.
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
constexpr int kTmemCols = 512;
constexpr int kABytes = kBW * 128;

__device__ int g_err;

struct GemmArgs {
  const uint8_t* wscales;
  const uint8_t* xscales;
  const float* wg;
  const float* xg;
  int64_t M, N;
  int wblocks, tblocks, kblocks;   // tiles of weight rows, of tokens, stages
  int kt, steps;                   // scale tiles along K, MMA steps of 64 columns
  int x_tiles;                     // scale tiles along the tokens
  const void* bias;
  int bias_dtype;
  void* out;
  int out_dtype;
  int64_t out_stride;
  int split;
  int* counters;
  float* partials;                 // split: [grid][2][128][BT]
  uint64_t wait_ns;
  int stall;                       // test hook: the producer issues nothing
};

template <bool NV, int BT>
struct Shape {
  static constexpr int kTiles = NV ? 4 : 2;                    // scale tiles of a stage, per 128 rows
  static constexpr int kXRowTiles = BT > 128 ? 2 : 1;
  static constexpr int kSfA = kTiles * kTileBytes;
  static constexpr int kSfB = kXRowTiles * kTiles * kTileBytes;
  static constexpr int kXBytes = BT * 128;
  static constexpr int kStage = kABytes + kXBytes + kSfA + kSfB;
  static constexpr int kSfCols = 4 * kTiles * (1 + kXRowTiles);  // TMEM columns of a stage's scales
  static constexpr int kAcc = BT <= 128 ? 2 : 1;               // accumulators
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

// Instruction descriptor: E2M1 operands, K-major, fp32 sums, M = 128 x N;
// sf: which of a column's scales the instruction starts from (mxfp4: 0 or 2).
template <bool NV>
__host__ __device__ constexpr uint32_t idesc_fp4(int N, uint32_t sf) {
  return (sf << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (NV ? 0u : 1u << 23) |
         ((uint32_t)(kBW >> 7) << 27) | (sf << 29);
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

// Work items of a CTA: a tile and the stages [k0, k1) of it that are its own.
struct Item {
  int tile, k0, k1, slot;
};
struct ItemIter {
  int64_t u, u1;
  int64_t begin;
};
__device__ __forceinline__ ItemIter items_begin(const GemmArgs& a, int ntiles) {
  ItemIter it;
  if (a.split) {
    const int64_t U = (int64_t)ntiles * a.kblocks;
    it.u = U * blockIdx.x / gridDim.x;
    it.u1 = U * (blockIdx.x + 1) / gridDim.x;
  } else {
    it.u = blockIdx.x;
    it.u1 = ntiles;
  }
  it.begin = it.u;
  return it;
}
__device__ __forceinline__ bool items_next(const GemmArgs& a, ItemIter& it, Item& x) {
  if (it.u >= it.u1) return false;
  if (a.split) {
    x.tile = (int)(it.u / a.kblocks);
    x.k0 = (int)(it.u - (int64_t)x.tile * a.kblocks);
    x.k1 = (int)min((int64_t)a.kblocks, x.k0 + (it.u1 - it.u));
    x.slot = it.u == it.begin ? 0 : 1;
    it.u += x.k1 - x.k0;
  } else {
    x.tile = (int)it.u;
    x.k0 = 0;
    x.k1 = a.kblocks;
    x.slot = 0;
    it.u += gridDim.x;
  }
  return true;
}

template <bool NV, int BT>
__global__ void __launch_bounds__(kThreads) fp4_gemm_kernel(const __grid_constant__ CUtensorMap wmap,
                                                            const __grid_constant__ CUtensorMap xmap,
                                                            const GemmArgs a) {
  using P = Shape<NV, BT>;
  constexpr int S = P::S;
  extern __shared__ char smem_raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  char* s_w = smem;                                  // [S][128][128]
  char* s_x = s_w + S * kABytes;                     // [S][BT][128]
  char* s_sw = s_x + S * P::kXBytes;                 // [S][tiles][512]
  char* s_sx = s_sw + S * P::kSfA;                   // [S][row tiles][tiles][512]
  uint64_t* full = reinterpret_cast<uint64_t*>(s_sx + S * P::kSfB);
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
    prefetch_tensormap(&xmap);
    for (int i = 0; i < S; ++i) {
      mbar_init(full + i, 1);
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
    if (lane == 0 && !a.stall) {
      int s = 0;
      uint32_t ph = 0;
      ItemIter it = items_begin(a, ntiles);
      Item x;
      bool ok = true;
      int issued = 0;
      while (ok && items_next(a, it, x)) {
        const int tb = x.tile % a.tblocks, wb = x.tile / a.tblocks;
        for (int kb = x.k0; kb < x.k1; ++kb) {
          if (!mbar_wait_hint(empty + s, ph ^ 1, &g_err, 21, a.wait_ns)) {
            ok = false;
            break;
          }
          const int t0 = kb * P::kTiles, nt = min(P::kTiles, a.kt - t0);
          const int xt = min(P::kXRowTiles, a.x_tiles - tb * P::kXRowTiles);   // (BT < 128 has one token tile)
          const uint32_t sf_bytes = nt * kTileBytes;
          mbar_arrive_expect_tx(full + s, kABytes + P::kXBytes + sf_bytes * (1 + xt));
          tma_load_2d(s_w + s * kABytes, &wmap, kb * 128, wb * kBW, full + s);
          tma_load_2d(s_x + s * P::kXBytes, &xmap, kb * 128, tb * BT, full + s);
          bulk_load(s_sw + s * P::kSfA, a.wscales + ((int64_t)wb * a.kt + t0) * kTileBytes, sf_bytes, full + s);
          for (int r = 0; r < xt; ++r)
            bulk_load(s_sx + s * P::kSfB + r * P::kSfA,
                      a.xscales + ((int64_t)(tb * P::kXRowTiles + r) * a.kt + t0) * kTileBytes, sf_bytes, full + s);
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
    if (lane == 0) {
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
            copy_scales(sfa + 4 * t, swd0 + (uint64_t)((s * P::kSfA + t * kTileBytes) >> 4));
#pragma unroll
            for (int r = 0; r < P::kXRowTiles; ++r)
              copy_scales(sfb + 4 * (t * P::kXRowTiles + r),
                          sxd0 + (uint64_t)((s * P::kSfB + r * P::kSfA + t * kTileBytes) >> 4));
          }
          const int nk = min(kBK / kColPad, a.steps - kb * (kBK / kColPad));
          const uint64_t wd = wd0 + (uint64_t)((s * kABytes) >> 4), xd = xd0 + (uint64_t)((s * P::kXBytes) >> 4);
          for (int k = 0; k < nk; ++k) {
            const int t = NV ? k : k >> 1;
            const uint32_t sf = NV ? 0u : (uint32_t)(k & 1) * 2;
            mma_fp4<NV>(d, wd + 2 * k, xd + 2 * k, idesc_fp4<NV>(BT, sf), sfa + 4 * t,
                        sfb + 4 * t * P::kXRowTiles, (kb != x.k0 || k != 0) ? 1u : 0u);
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
  } else {
    const int quad = warp & 3;
    const int r = quad * 32 + lane;                  // this thread's row of the tile
    const float alpha = usable_scale(a.wg) * usable_scale(a.xg);
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
      float* pp = whole ? nullptr : a.partials + ((size_t)blockIdx.x * 2 + x.slot) * (BT * kBW);
      const float bias = a.bias && valid ? load_f(a.bias, a.bias_dtype, n) : 0.f;
      const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + buf * P::kAccCols;
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
          float4* dst = reinterpret_cast<float4*>(pp + (size_t)r * BT + c * CW);
#pragma unroll
          for (int j = 0; j < CW / 4; ++j) dst[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          continue;
        }
        if (!valid) continue;
        const int64_t mb = m0 + c * CW;
        const int jn = (int)min((int64_t)CW, a.M - mb);
#pragma unroll
        for (int j = 0; j < CW; ++j)
          if (j < jn) store_f(a.out, a.out_dtype, (mb + j) * a.out_stride + n, fmaf(v[j], alpha, bias));
      }
      if (++buf == P::kAcc) {
        buf = 0;
        bph ^= 1;
      }
      if (whole) continue;
      // a tile split over several CTAs: the last to arrive adds the pieces
      __threadfence();
      named_bar_sync(3, kEpiWarps * 32);
      if (r == 0) *epi_flag = atomicAdd(a.counters + x.tile, 1);
      named_bar_sync(3, kEpiWarps * 32);
      const int64_t U = (int64_t)ntiles * a.kblocks;
      const int G = gridDim.x;
      const int64_t u_lo = (int64_t)x.tile * a.kblocks, u_hi = u_lo + a.kblocks - 1;
      const int c_first = (int)(((u_lo + 1) * G - 1) / U), c_last = (int)(((u_hi + 1) * G - 1) / U);
      const int old = *epi_flag;
      named_bar_sync(3, kEpiWarps * 32);
      if (old != c_last - c_first) continue;
      __threadfence();
      if (r == 0) a.counters[x.tile] = 0;
      if (!valid) continue;
      constexpr int RT = 16;
      for (int j0 = 0; j0 < jn_all; j0 += RT) {
        float sum[RT];
#pragma unroll
        for (int u = 0; u < RT; ++u) sum[u] = 0.f;
        for (int c = c_first; c <= c_last; ++c) {
          const int slot = U * c / G >= u_lo ? 0 : 1;
          const float4* src =
              reinterpret_cast<const float4*>(a.partials + ((size_t)c * 2 + slot) * (BT * kBW) + (size_t)r * BT + j0);
          float4 t[RT / 4];
#pragma unroll
          for (int u = 0; u < RT / 4; ++u) t[u] = __ldcg(src + u);
#pragma unroll
          for (int u = 0; u < RT / 4; ++u) {
            sum[4 * u] += t[u].x;
            sum[4 * u + 1] += t[u].y;
            sum[4 * u + 2] += t[u].z;
            sum[4 * u + 3] += t[u].w;
          }
        }
#pragma unroll
        for (int u = 0; u < RT; ++u)
          if (j0 + u < jn_all)
            store_f(a.out, a.out_dtype, (m0 + j0 + u) * a.out_stride + n, fmaf(sum[u], alpha, bias));
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ---- host -------------------------------------------------------------------

struct Plan {
  int BT, tblocks, wblocks, kblocks, ntiles, grid;
  bool split;
};

static Plan plan(int64_t M, int64_t N, int64_t K) {
  Plan p;
  p.BT = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : M <= 128 ? 128 : 256;
  p.wblocks = (int)((N + kBW - 1) / kBW);
  p.tblocks = (int)((M + p.BT - 1) / p.BT);
  p.kblocks = (int)((padded_cols(K) + kBK - 1) / kBK);
  p.ntiles = p.wblocks * p.tblocks;
  p.split = p.BT <= 128;
  p.grid = (int)std::min<int64_t>(p.split ? (int64_t)p.ntiles * p.kblocks : p.ntiles, sm_count());
  return p;
}

template <bool NV, int BT>
static int launch(const CUtensorMap& wm, const CUtensorMap& xm, const GemmArgs& a, int grid, cudaStream_t st) {
  auto k = fp4_gemm_kernel<NV, BT>;
  constexpr size_t smem = Shape<NV, BT>::kSmem;
  static_assert(smem <= 227 * 1024, "shared memory");
  static thread_local int configured_dev = -1;
  int dev = 0;
  TS_CUDA_TRY(cudaGetDevice(&dev));
  if (configured_dev != dev) {
    TS_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    configured_dev = dev;
  }
  k<<<grid, kThreads, smem, st>>>(wm, xm, a);
  TS_LAUNCH_CHECK();
  return TS_OK;
}

template <bool NV>
static int launch(int BT, const CUtensorMap& wm, const CUtensorMap& xm, const GemmArgs& a, int grid, cudaStream_t st) {
  switch (BT) {
    case 16: return launch<NV, 16>(wm, xm, a, grid, st);
    case 32: return launch<NV, 32>(wm, xm, a, grid, st);
    case 64: return launch<NV, 64>(wm, xm, a, grid, st);
    case 128: return launch<NV, 128>(wm, xm, a, grid, st);
    default: return launch<NV, 256>(wm, xm, a, grid, st);
  }
}

}  // namespace fp4

}  // namespace ts

using namespace ts;
using namespace ts::fp4;

extern "C" size_t ts_fp4_matmul_workspace_size(int64_t M, int64_t N, int64_t K, int format) {
  (void)format;
  if (M <= 0 || N <= 0 || K <= 0) return paged::kCounterBytes;
  const Plan p = plan(M, N, K);
  return paged::kCounterBytes + (p.split ? (size_t)p.grid * 2 * kBW * p.BT * 4 : 0);
}

extern "C" int ts_fp4_matmul(const ts_fp4_tensor* x, const ts_fp4_tensor* w, const void* bias, int bias_dtype, void* out,
                             int out_dtype, int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                             void* stream) {
  int rc = check_tensor(x, "ts_fp4_matmul a");
  if (rc != TS_OK) return rc;
  rc = check_tensor(w, "ts_fp4_matmul b");
  if (rc != TS_OK) return rc;
  TS_REQUIRE(x->format == w->format, "both operands must have one format");
  TS_REQUIRE(x->cols == w->cols, "a has %lld columns, b %lld", (long long)x->cols, (long long)w->cols);
  TS_UNSUPPORTED(out_dtype == TS_F16 || out_dtype == TS_BF16 || out_dtype == TS_F32, "unknown output type %d", out_dtype);
  TS_UNSUPPORTED(!bias || bias_dtype == TS_F16 || bias_dtype == TS_BF16 || bias_dtype == TS_F32, "unknown bias type %d",
                 bias_dtype);
  if (x->rows == 0 || w->rows == 0) return TS_OK;
  TS_REQUIRE(out, "NULL pointer");
  const Plan p = plan(x->rows, w->rows, w->cols);
  const size_t need = ts_fp4_matmul_workspace_size(x->rows, w->rows, w->cols, w->format);
  if (p.split && (workspace == nullptr || workspace_bytes < need)) {
    set_error("workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return TS_ERR_WORKSPACE;
  }
  TS_REQUIRE(is_aligned(workspace, 16), "workspace must be 16-byte aligned");
  TS_UNSUPPORTED(!p.split || p.ntiles <= (int)paged::kCounters, "too many output features in one call");
  GemmArgs a;
  a.wscales = w->scales;
  a.xscales = x->scales;
  a.wg = w->format == TS_NVFP4 ? w->global_scale : nullptr;
  a.xg = x->format == TS_NVFP4 ? x->global_scale : nullptr;
  a.M = x->rows;
  a.N = w->rows;
  a.wblocks = p.wblocks;
  a.tblocks = p.tblocks;
  a.kblocks = p.kblocks;
  a.kt = (int)scale_tiles(w->cols, w->format);
  a.steps = (int)(padded_cols(w->cols) / kColPad);
  a.x_tiles = (int)((x->rows + kTileRows - 1) / kTileRows);
  a.bias = bias;
  a.bias_dtype = bias_dtype;
  a.out = out;
  a.out_dtype = out_dtype;
  a.out_stride = out_row_stride;
  a.split = p.split ? 1 : 0;
  a.counters = reinterpret_cast<int*>(workspace);
  a.partials = p.split ? reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + paged::kCounterBytes) : nullptr;
  a.wait_ns = wait_limit_ns();
  a.stall = take_test_stall() ? 1 : 0;
  const uint64_t row = (uint64_t)padded_cols(w->cols) / 2;
  CUtensorMap wm, xm;
  rc = encode_tmap_2d(&wm, w->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, row, (uint64_t)w->rows, row, 128, kBW,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != TS_OK) return rc;
  rc = encode_tmap_2d(&xm, x->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, row, (uint64_t)x->rows, row, 128, p.BT,
                      CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != TS_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return w->format == TS_NVFP4 ? launch<true>(p.BT, wm, xm, a, p.grid, st) : launch<false>(p.BT, wm, xm, a, p.grid, st);
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
  const size_t need = ts_fp4_linear_workspace_size(M, w->rows, w->cols, w->format);
  if (workspace == nullptr || workspace_bytes < need) {
    set_error("workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return TS_ERR_WORKSPACE;
  }
  TS_REQUIRE(is_aligned(workspace, 16), "workspace must be 16-byte aligned");
  // the activations' codes and scales lie behind the product's scratch
  const size_t at = align_up(ts_fp4_matmul_workspace_size(M, w->rows, w->cols, w->format), 256);
  ts_fp4_tensor t{};
  t.codes = reinterpret_cast<uint8_t*>(workspace) + at;
  t.scales = t.codes + align_up((size_t)M * (size_t)(padded_cols(w->cols) / 2), 256);
  t.global_scale = w->format == TS_NVFP4 ? x_scale : nullptr;
  t.rows = M;
  t.cols = w->cols;
  t.format = w->format;
  rc = ts_fp4_quantize(x, x_dtype, x_row_stride, &t, 0, nullptr, 0, stream);
  if (rc != TS_OK) return rc;
  return ts_fp4_matmul(&t, w, bias, bias_dtype, out, out_dtype, out_row_stride, workspace, at, stream);
}
