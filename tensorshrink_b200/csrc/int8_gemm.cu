// Product of two matrices of 8-bit integers with a scale per row of each.
//
//   out[m, n] = s_m t_n sum_k qa[m, k] qb[n, k] (+ bias[n])
//
// tcgen05.mma kind::i8 with 32-bit integer sums: they are exact, whatever the
// order or the split, and the result is rounded when a sum becomes fp32, at each of
// the two products with a scale, at the bias, and to the output's type.
//
// Two kernels: int8_gemm_kernel for decode-sized calls and small layers,
// int8_pair_kernel (below) for prefill.
//
// int8_gemm_kernel: a tile is 128 rows of b (the weight's output features; the
// MMA's M) x BT <= 128 rows of a (tokens; its N), K in stages of 128. Roles in
// one persistent CTA per SM:
//   warp 0      TMA producer: codes of both operands, rows of 128 bytes with the
//               128-byte swizzle
//   warp 1      one thread issues the MMAs
//   warps 2-5   epilogue: tcgen05.ld, scales, bias, stores
//   warps 6-13  (kernels of few tokens that come unquantised) find the tokens' scales and
//               quantise the stages' columns into shared memory, a stage per warp in turn
// Bound by the weight's bytes. The tiles are few, so they are split along K:
// into whole parts, whose CTAs are a cluster and add their sums through
// distributed shared memory, or, where clusters do not fit the tiles, into
// equal shares of all stages laid end to end, whose sums the last CTA of a
// tile to arrive adds from the workspace. Measured, other weights each call: 14336 x
// 4096, 1 token 11.6 us (13.6 with its quantisation), 4096 x 14336, 33 tokens 14.3 (59 MB, 9.0 us at the copy
// bandwidth; the rest is start, first loads and epilogue).
//
// Every wait is bounded in wall-clock time: a role whose wait runs out records
// a code and unwinds; the TMEM is freed at the end in any case.
#include <algorithm>

#include "gemm.cuh"
#include "int8.cuh"
#include "paged.cuh"

namespace ts {
namespace int8 {

constexpr int kBW = 128;                 // weight rows of a tile = TMEM lanes
constexpr int kBK = 128;                 // columns of a stage = one 128-byte row
constexpr int kStep = 32;                // columns of an MMA
constexpr int kEpiWarps = 4;
constexpr int kThreads = (2 + kEpiWarps) * 32;
constexpr int kABytes = kBW * kBK;
constexpr int kMaxCluster = 8;           // CTAs of a cluster that share a tile
constexpr int kQuantWarps = 8;

// Up to this many tokens, of this many elements together, the kernel quantises them itself:
// every CTA finds their scales (each reads all of them, from L2) while its first weights
// are on their way. More come from a quantiser in front, which the kernel's start
// overlaps. 14336 x 4096: one token 13.6 us by itself, 14.7 behind a quantiser, two
// 14.3 and 14.6, four 16.1 and 14.8; 8192 x 28672, one token 47.3 and 44.5.
constexpr int kOwnTokens = 2;
constexpr int64_t kOwnElements = 16384;

__device__ int g_err;

struct GemmArgs {
  const float* wscales;
  const float* xscales;
  int64_t M, N;
  int wblocks, tblocks, kblocks;   // tiles of weight rows, of tokens, stages
  int steps;                       // MMA steps of 32 columns
  const void* bias;
  int bias_dtype;
  void* out;
  int out_dtype;
  int64_t out_stride;
  int* counters;                   // one per tile, zero between calls
  int* partials;                   // [grid][2][BT / 4][128][4]
  uint64_t wait_ns;
  int stall;                       // test hook: the producer issues nothing
  int cluster;                     // CTAs that share a tile as a cluster, or 0
  int out_vec;                     // rows of out take stores of four values
  const void* x;                   // tokens to be quantised by the kernel itself
  int x_dtype, x_aligned;          // x_aligned: rows start on 16 bytes
  int64_t x_stride, K;
};

template <int BT>
struct Shape {
  static constexpr int kXBytes = BT * kBK;
  static constexpr int kStage = kABytes + kXBytes;
  static constexpr int kAcc = 2;                               // accumulators
  static constexpr int kAccCols = BT < 32 ? 32 : BT;
  static constexpr int kTmem = kAcc * kAccCols;
  static constexpr int kFit = (227 * 1024 - 2048 - BT * 4) / kStage;
  static constexpr int S = kFit < 12 ? kFit : 12;
  static constexpr size_t kSmem = 1024 + (size_t)S * kStage + (2 * S + 2 * kAcc + 1) * 8 + 16 + BT * 4;
};

// Instruction descriptor: signed 8-bit operands, K-major, 32-bit integer sums, M x N.
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// sum s t + bias, by the smaller scale first: with a scale of at least 2^-100
// that product keeps clear of the range's lower end, and it passes the upper
// one only where the result does. A NaN of either scale stays.
__device__ __forceinline__ float scaled(int sum, float s, float t, float bias) {
  float lo, hi;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(lo) : "f"(s), "f"(t));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(hi) : "f"(s), "f"(t));
  return __fadd_rn(__fmul_rn(__fmul_rn((float)sum, lo), hi), bias);
}

// Stores the results of `jn` tokens from m on, of output feature n (one per
// lane: the lanes of a warp store neighbours).
template <int R>
__device__ __forceinline__ void store_tokens(const GemmArgs& a, int64_t m, int64_t n, int jn, const int* v, const float* xs,
                                             float ws, float bias) {
  const int64_t at = m * a.out_stride + n, step = a.out_stride;
  if (a.out_dtype == TS_F32) {
    float* p = reinterpret_cast<float*>(a.out) + at;
#pragma unroll
    for (int j = 0; j < R; ++j, p += step)
      if (j < jn) *p = scaled(v[j], xs[j], ws, bias);
  } else if (a.out_dtype == TS_BF16) {
    __nv_bfloat16* p = reinterpret_cast<__nv_bfloat16*>(a.out) + at;
#pragma unroll
    for (int j = 0; j < R; ++j, p += step)
      if (j < jn) *p = __float2bfloat16_rn(scaled(v[j], xs[j], ws, bias));
  } else {
    __half* p = reinterpret_cast<__half*>(a.out) + at;
#pragma unroll
    for (int j = 0; j < R; ++j, p += step)
      if (j < jn) *p = __float2half_rn(scaled(v[j], xs[j], ws, bias));
  }
}

// Stores the results of output features n .. n + 3 of token m.
__device__ __forceinline__ void store_four(const GemmArgs& a, int64_t m, int64_t n, const int (&v)[4], float xs) {
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool has = n + i < a.N;
    f[i] = scaled(v[i], xs, has ? a.wscales[n + i] : 0.f, a.bias && has ? load_f(a.bias, a.bias_dtype, n + i) : 0.f);
  }
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
  const bool bf = a.out_dtype == TS_BF16;
  const uint2 w = bf ? make_uint2(paged::pack2<true>(f[0], f[1]), paged::pack2<true>(f[2], f[3]))
                     : make_uint2(paged::pack2<false>(f[0], f[1]), paged::pack2<false>(f[2], f[3]));
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
struct Items {
  int64_t u, u1;
  __device__ __forceinline__ Items(const GemmArgs& a, int ntiles) {
    const int64_t all = (int64_t)ntiles * a.kblocks;
    u = all * blockIdx.x / gridDim.x;
    u1 = all * (blockIdx.x + 1) / gridDim.x;
  }
  __device__ __forceinline__ bool next(const GemmArgs& a, Item& x) {
    if (u >= u1) return false;
    x.tile = (int)(u / a.kblocks);
    x.k0 = (int)(u - (int64_t)x.tile * a.kblocks);
    x.k1 = (int)min((int64_t)a.kblocks, x.k0 + (u1 - u));
    u += x.k1 - x.k0;
    return true;
  }
};

// By the quantising warps: the scales of all tokens to xs[] (and to r[] their inverses, 0
// of a token that is not finite).
template <int DT>
__device__ __forceinline__ void token_scales(const GemmArgs& a, float* xs, float* r, uint32_t (*tops)[kOwnTokens]) {
  using T = typename Elem<DT>::T;
  const int t = threadIdx.x - kThreads, warp = t >> 5, chunks = (int)((a.K + 7) / 8), M = (int)a.M;
  for (int m = 0; m < M; ++m) {
    const T* row = reinterpret_cast<const T*>(a.x) + m * a.x_stride;
    uint32_t top = 0;
    constexpr int kAhead = 4, N = DT == TS_F32 ? 8 : 4;
    for (int c = t; c < chunks; c += kAhead * kQuantWarps * 32) {
      uint32_t w[kAhead][N];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int ci = c + i * kQuantWarps * 32;
        const int64_t cols = ci < chunks ? a.K : 0;      // (nothing is loaded behind the last column)
        if (a.x_aligned) load8<DT, true>(row, ci, cols, w[i]);
        else load8<DT, false>(row, ci, cols, w[i]);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) top = max(top, top8<DT>(w[i]));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((t & 31) == 0) tops[warp][m] = top;
  }
  named_bar_sync(4, kQuantWarps * 32);
  if (t < M) {
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < kQuantWarps; ++w) top = max(top, tops[w][t]);
    const bool finite = top < 0x7F800000u;
    const float s = finite ? scale_of(__uint_as_float(top)) : __uint_as_float(0x7FC00000u);
    xs[t] = s;
    r[t] = finite ? __frcp_rn(s) : 0.f;
  }
  named_bar_sync(4, kQuantWarps * 32);
}

// Columns [128 kb, 128 kb + 128) of all tokens into a stage, as TMA would swizzle them: 16 lanes a
// row, eight columns each.
template <int DT>
__device__ __forceinline__ void quantise_stage(const GemmArgs& a, int kb, char* sx, const float* r) {
  using T = typename Elem<DT>::T;
  const int lane = threadIdx.x & 31, j = lane & 15;
  for (int m = lane >> 4; m < a.M; m += 2) {
    const T* row = reinterpret_cast<const T*>(a.x) + m * a.x_stride;
    uint32_t w[DT == TS_F32 ? 8 : 4];
    if (a.x_aligned) load8<DT, true>(row, kb * 16 + j, a.K, w);
    else load8<DT, false>(row, kb * 16 + j, a.K, w);
    const float f = r[m];
    *reinterpret_cast<uint2*>(sx + m * 128 + (((j >> 1) ^ (m & 7)) << 4) + (j & 1) * 8) =
        f != 0.f ? codes8<DT>(w, f) : make_uint2(0, 0);
  }
}

template <int BT, bool Q>
__global__ void __launch_bounds__(kThreads + (Q ? kQuantWarps * 32 : 0), 1)
int8_gemm_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const GemmArgs a) {
  using P = Shape<BT>;
  constexpr int S = P::S;
  static_assert(!Q || BT >= kOwnTokens, "tokens of a stage");
  __shared__ uint32_t q_tops[kQuantWarps][kOwnTokens];
  __shared__ float q_inv[kOwnTokens];
  extern __shared__ char smem_raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  char* s_w = smem;                                  // [S][128][128]
  char* s_x = s_w + S * kABytes;                     // [S][BT][128]
  uint64_t* full = reinterpret_cast<uint64_t*>(s_x + S * P::kXBytes);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + P::kAcc;
  uint64_t* drain = tempty + P::kAcc;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  int* epi_flag = reinterpret_cast<int*>(tmem_slot + 1);
  float* s_xs = reinterpret_cast<float*>(tmem_slot + 4);   // [BT] the tile's token scales

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
    tmem_alloc(tmem_slot, P::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      auto load_w = [&](const Item& x, int kb, int s) {
        mbar_arrive_expect_tx(full + s, Q ? kABytes : P::kStage);
        tma_load_2d(s_w + s * kABytes, &wmap, kb * kBK, x.tile / a.tblocks * kBW, full + s);
      };
      // The weight's first S stages are loaded while the kernel that writes
      // the tokens' codes may still run; everything else follows its end.
      Items it(a, ntiles);
      const int ahead = a.stall ? 0 : (int)min((int64_t)S, it.u1 - it.u);
      int s = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = !a.stall;
      Item x;
      while (issued < ahead && it.next(a, x))
        for (int kb = x.k0; kb < x.k1 && issued < ahead; ++kb) load_w(x, kb, issued++);
      pdl_wait_primary();
      issued = 0;
      it = Items(a, ntiles);
      while (ok && it.next(a, x)) {
        for (int kb = x.k0; kb < x.k1; ++kb) {
          if (issued >= ahead) {
            if (!mbar_wait_hint(empty + s, ph ^ 1, &g_err, 41, a.wait_ns)) {
              ok = false;
              break;
            }
            load_w(x, kb, s);
          }
          if (!Q) tma_load_2d(s_x + s * P::kXBytes, &xmap, kb * kBK, x.tile % a.tblocks * BT, full + s);
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
      int s = 0, buf = 0;
      uint32_t ph = 0, bph = 0;
      Items it(a, ntiles);
      Item x;
      bool ok = true;
      while (ok && it.next(a, x)) {
        if (!mbar_wait_hint(tempty + buf, bph ^ 1, &g_err, 42, a.wait_ns)) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * P::kAccCols;
        for (int kb = x.k0; kb < x.k1; ++kb) {
          if (!mbar_wait_hint(full + s, ph, &g_err, 43, a.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int nk = min(kBK / kStep, a.steps - kb * (kBK / kStep));
          const uint64_t wd = wd0 + (uint64_t)((s * kABytes) >> 4), xd = xd0 + (uint64_t)((s * P::kXBytes) >> 4);
          for (int k = 0; k < nk; ++k)
            mma_i8(d, wd + 2 * k, xd + 2 * k, idesc_i8(kBW, BT), (kb != x.k0 || k != 0) ? 1u : 0u);
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
    if (a.x_dtype == TS_BF16) token_scales<TS_BF16>(a, s_xs, q_inv, q_tops);
    else if (a.x_dtype == TS_F16) token_scales<TS_F16>(a, s_xs, q_inv, q_tops);
    else token_scales<TS_F32>(a, s_xs, q_inv, q_tops);
    int n = 0;                                       // of the CTA's stages
    bool ok = true;
    Items it(a, ntiles);
    Item x;
    while (ok && it.next(a, x)) {
      for (int kb = x.k0; kb < x.k1; ++kb, ++n) {
        if (n % kQuantWarps != warp - (2 + kEpiWarps)) continue;
        const int s = n % S;
        ok = __all_sync(0xffffffffu, mbar_wait_hint(empty + s, (uint32_t)(n / S & 1) ^ 1, &g_err, 45, a.wait_ns));
        if (!ok) break;
        char* sx = s_x + s * P::kXBytes;
        if (a.x_dtype == TS_BF16) quantise_stage<TS_BF16>(a, kb, sx, q_inv);
        else if (a.x_dtype == TS_F16) quantise_stage<TS_F16>(a, kb, sx, q_inv);
        else quantise_stage<TS_F32>(a, kb, sx, q_inv);
        fence_proxy_async_smem();                    // the tensor cores read what was written
        __syncwarp();
        if (lane == 0) mbar_arrive(full + s);
      }
    }
  } else {
    const int quad = warp & 3;
    const int r = quad * 32 + lane;                  // this thread's row of the tile
    constexpr int CW = BT < 32 ? 16 : 32;
    int buf = 0;
    uint32_t bph = 0;
    Items it(a, ntiles);
    Item x;
    pdl_wait_primary();                              // (the token scales)
    while (it.next(a, x)) {
      const int64_t m0 = (int64_t)(x.tile % a.tblocks) * BT;
      const int64_t n = (int64_t)(x.tile / a.tblocks) * kBW + r;
      const int jn_all = (int)min((int64_t)BT, a.M - m0);
      const bool valid = n < a.N;
      named_bar_sync(3, kEpiWarps * 32);             // (the last tile's scales have been used)
      if (!Q && r < jn_all) s_xs[r] = a.xscales[m0 + r];   // (else its quantisers have put them there)
      const float ws = valid ? a.wscales[n] : 0.f;
      const float bias = a.bias && valid ? load_f(a.bias, a.bias_dtype, n) : 0.f;
      if (!named_bar_and(3, kEpiWarps * 32, mbar_wait_hint(tfull + buf, bph, &g_err, 44, a.wait_ns))) break;
      tc_fence_after();
      const bool whole = x.k0 == 0 && x.k1 == a.kblocks;
      int* pp = whole ? nullptr : a.partials + ((size_t)blockIdx.x * 2 + (x.k0 > 0 ? 0 : 1)) * (BT * kBW);
      const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + buf * P::kAccCols;
      auto load = [&](int c, int (&v)[CW]) {
        float f[CW];
        if constexpr (CW == 32) tmem_ld32(acc + c * CW, f);
        else tmem_ld16(acc + c * CW, f);
#pragma unroll
        for (int j = 0; j < CW; ++j) v[j] = __float_as_int(f[j]);
      };
      if (a.cluster) {
        // to shared memory, over the stages (all used): [BT tokens][128 rows]
        // (the CTA's only item: nobody waits for the accumulator)
#pragma unroll 1
        for (int c = 0; c < BT / CW && c * CW < jn_all; ++c) {
          int v[CW];
          load(c, v);
          int* dst = reinterpret_cast<int*>(s_w) + c * CW * kBW + r;
#pragma unroll
          for (int j = 0; j < CW; ++j) dst[j * kBW] = v[j];
        }
        break;
      }
#pragma unroll 1
      for (int c = 0; c < BT / CW; ++c) {
        int v[CW];
        load(c, v);
        if (c == BT / CW - 1) {
          tc_fence_before();
          mbar_arrive(tempty + buf);
        }
        if (!whole) {
          // a piece: [BT / 4 tokens][128 rows][4 tokens], coalesced both ways
          int4* dst = reinterpret_cast<int4*>(pp) + (size_t)(c * CW / 4) * kBW + r;
#pragma unroll
          for (int j = 0; j < CW / 4; ++j)
            if (c * CW + 4 * j < jn_all) dst[j * kBW] = make_int4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          continue;
        }
        if (!valid) continue;
        store_tokens<CW>(a, m0 + c * CW, n, min(CW, jn_all - c * CW), v, s_xs + c * CW, ws, bias);
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
      if (*epi_flag != c_last - c_first) continue;     // (rewritten behind the next item's barriers)
      if (r == 0) a.counters[x.tile] = 0;
      if (!valid) continue;
      // the tile's beginning lies in its CTA's second slot, the other pieces
      // in their CTAs' first; kRun tokens of 4 pieces in flight
      constexpr int kPiece4 = BT * kBW / 4;
      const int4* base = reinterpret_cast<const int4*>(a.partials) + (size_t)c_first * 2 * kPiece4 + r;
      const int pieces = c_last - c_first + 1;
      constexpr int kRun = BT < 32 ? BT : 32, kRun4 = kRun / 4;   // tokens of a round
      for (int j0 = 0; j0 < jn_all; j0 += kRun) {
        int sum[kRun];
#pragma unroll
        for (int u = 0; u < kRun; ++u) sum[u] = 0;
        for (int c = 0; c < pieces; c += 4) {
          // (tokens behind the last one were not written: read, never stored)
          int4 t[4][kRun4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int cc = min(c + i, pieces - 1);
            const int4* src = base + (cc == 0 ? (size_t)kPiece4 : (size_t)cc * 2 * kPiece4) + (size_t)(j0 / 4) * kBW;
#pragma unroll
            for (int u = 0; u < kRun4; ++u) t[i][u] = __ldcg(src + u * kBW);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (c + i >= pieces) break;
#pragma unroll
            for (int u = 0; u < kRun4; ++u) {
              sum[4 * u] += t[i][u].x;
              sum[4 * u + 1] += t[i][u].y;
              sum[4 * u + 2] += t[i][u].z;
              sum[4 * u + 3] += t[i][u].w;
            }
          }
        }
        store_tokens<kRun>(a, m0 + j0, n, min(kRun, jn_all - j0), sum, s_xs + j0, ws, bias);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, P::kTmem);
  }
  if (a.cluster) {
    // every CTA of the tile has its sums in shared memory: a warp adds a
    // token's, four neighbouring features per lane
    static_assert((size_t)BT * kBW * 4 <= (size_t)S * kABytes, "the sums lie over the stages");
    cluster_sync();
    pdl_wait_primary();
    const int rank = (int)cta_rank(), tile = blockIdx.x / a.cluster;
    const int64_t m0 = (int64_t)(tile % a.tblocks) * BT, n = (int64_t)(tile / a.tblocks) * kBW + 4 * lane;
    const int jn = (int)min((int64_t)BT, a.M - m0);
    constexpr int kWarpsAll = kThreads / 32 + (Q ? kQuantWarps : 0);
    for (int j = rank + a.cluster * warp; j < jn; j += a.cluster * kWarpsAll) {
      const uint32_t at = smem_u32(s_w) + (uint32_t)(j * kBW + 4 * lane) * 4;
      float4 v[kMaxCluster];
#pragma unroll
      for (int p = 0; p < kMaxCluster; ++p)
        if (p < a.cluster) v[p] = ld_cluster(map_cta(at, p));
      int sum[4] = {0, 0, 0, 0};
#pragma unroll
      for (int p = 0; p < kMaxCluster; ++p)
        if (p < a.cluster) {
          sum[0] += __float_as_int(v[p].x);
          sum[1] += __float_as_int(v[p].y);
          sum[2] += __float_as_int(v[p].z);
          sum[3] += __float_as_int(v[p].w);
        }
      if (n < a.N) store_four(a, m0 + j, n, sum, Q ? s_xs[j] : a.xscales[m0 + j]);
    }
    cluster_sync();                                    // nobody leaves while its sums may be read
  }
}

// ---- prefill: tiles of 256 tokens x BN <= 256 weight rows on CTA pairs ------------
//
// Two CTAs of a cluster share one MMA (cta_group::2, M = 256): each holds its
// 128 token rows of A, half of B's rows and the accumulator of its own tokens, so
// that every operand byte is fetched by one of the two and feeds both tensor
// cores. Loads of both CTAs complete on the leader's barrier; the leader's
// thread issues the MMAs for both; commits release the stage in both. Tokens are
// the accumulator's lanes, so that a thread stores runs of its token's outputs.
// Two accumulators: a tile's epilogue runs under the next one's products. BN is chosen so
// that the tiles come out as few rounds of all pairs as their size allows. Measured: 8191 x 28672 x
// 8192 1.17 to 1.25 ms, 3.1 to 3.3 POP/s at the power limit (1.4 GHz, 92% of the tensor pipe's cycles);
// 2047 x 14336 x 4096 81 us, 3.0 POP/s; 256 x 4096 x 4096 9.9 us.

constexpr int kPairEpi = 8, kPairThreads = (2 + kPairEpi) * 32;
constexpr int kOutWords = 32 * 17;         // an epilogue warp's staging: 32 rows of 16 words, one word apart

template <int BN>
struct Pair {
  static constexpr int kHalf = BN / 2;                         // columns of an epilogue warp, B's rows of a CTA
  static constexpr int kBBytes = BN / 2 * kBK;
  static constexpr int kStage = kABytes + kBBytes;
  static constexpr int kAcc = 2;
  static constexpr int kAccCols = 256;                          // tensor memory comes in powers of two
  static constexpr int kEpi = 256 + kPairEpi * (2 * kHalf + kOutWords) * 4;   // barriers, then the epilogue warps' words
  static constexpr int kFit = (227 * 1024 - 1024 - kEpi) / kStage;
  static constexpr int S = kFit < 10 ? kFit : 10;
  static_assert((2 * S + 2 * kAcc + 1) * 8 + 4 <= 256, "barriers");
  static constexpr size_t kSmem = 1024 + (size_t)S * kStage + kEpi;
};

struct PairArgs {
  const float* wscales;
  const float* xscales;
  int64_t M, N;
  int mblocks, nblocks, kblocks;
  int group;                       // token blocks that are taken through all weight rows together
  int steps;
  const void* bias;
  int bias_dtype;
  void* out;
  int out_dtype;
  int64_t out_stride;
  int vec;                         // rows of out take 16-byte stores
  uint64_t wait_ns;
  int stall;
};

// Tile -> blocks of tokens and of weight rows: `group` token blocks at a time, the
// tokens running fastest, so that what the pairs read together, and the group's tokens over all
// rounds, stay in each half of L2 (8191 x 28672 x 8192 in one group of all 32: 1.9 GB from DRAM).
__device__ __forceinline__ void tile_at(const PairArgs& a, int tile, int* mb, int* nb) {
  const int g = tile / (a.group * a.nblocks), r = tile - g * a.group * a.nblocks;
  const int wide = min(a.group, a.mblocks - g * a.group);
  *nb = r / wide;
  *mb = g * a.group + r - *nb * wide;
}

template <int BN>
__global__ void __launch_bounds__(kPairThreads, 1) __cluster_dims__(2, 1, 1)
    int8_pair_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap, const PairArgs a) {
  using P = Pair<BN>;
  constexpr int S = P::S, kHalf = P::kHalf;
  extern __shared__ char smem_raw[];
  // both CTAs have one layout: the dynamic area starts at the same address in each
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  char* s_a = smem;
  char* s_b = s_a + S * kABytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(s_b + S * P::kBBytes);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + P::kAcc;
  uint64_t* drain = tempty + P::kAcc;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  char* s_epi = reinterpret_cast<char*>(full) + 256;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int ntiles = a.mblocks * a.nblocks;
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&amap);
    prefetch_tensormap(&bmap);
    for (int i = 0; i < S; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < P::kAcc; ++i) {
      mbar_init(tfull + i, 1);
      mbar_init(tempty + i, 2 * kPairEpi);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(P::kAcc * P::kAccCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      // Both CTAs' copies count on the leader's barrier. The first stages' weights are loaded
      // while the kernel that writes the tokens' codes may still run; everything
      // else follows its end.
      const int ahead = a.stall ? 0 : min(S, a.kblocks);     // (a pair has at least one tile)
      int mb, nb;
      tile_at(a, pair, &mb, &nb);
      const int brow0 = nb * BN + (int)rank * (BN / 2), arow0 = mb * 256 + (int)rank * 128;
      for (int kb = 0; kb < ahead; ++kb) {
        if (rank == 0) mbar_arrive_expect_tx(full + kb, 2 * P::kStage);
        tma_load_pair(smem_u32(s_b + kb * P::kBBytes), &bmap, kb * kBK, brow0, map_cta(smem_u32(full + kb), 0));
      }
      pdl_wait_primary();
      for (int kb = 0; kb < ahead; ++kb)
        tma_load_pair(smem_u32(s_a + kb * kABytes), &amap, kb * kBK, arow0,
                      map_cta(smem_u32(full + kb), 0));
      int s = ahead == S ? 0 : ahead, kb = ahead;
      uint32_t ph = ahead == S ? 1 : 0;
      bool ok = !a.stall;
      for (int tile = pair; ok && tile < ntiles; tile += pairs, kb = 0) {
        tile_at(a, tile, &mb, &nb);
        const int arow = mb * 256 + (int)rank * 128, brow = nb * BN + (int)rank * (BN / 2);
        for (; kb < a.kblocks; ++kb) {
          if (!mbar_wait_hint(empty + s, ph ^ 1, &g_err, 51, a.wait_ns)) {
            ok = false;
            break;
          }
          const uint32_t bar = map_cta(smem_u32(full + s), 0);
          if (rank == 0) mbar_arrive_expect_tx(full + s, 2 * P::kStage);
          tma_load_pair(smem_u32(s_a + s * kABytes), &amap, kb * kBK, arow, bar);
          tma_load_pair(smem_u32(s_b + s * P::kBBytes), &bmap, kb * kBK, brow, bar);
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      // every stage has been released to this CTA before it ends; after a
      // timeout, the copies in flight have landed
      for (int i = 0; i < S && !a.stall; ++i) {
        if (ok) {
          if (!mbar_wait_hint(empty + s, ph ^ 1, &g_err, 55, a.wait_ns)) break;
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
      int s = 0, buf = 0;
      uint32_t ph = 0, bph = 0;
      bool ok = true;
      for (int tile = pair; ok && tile < ntiles; tile += pairs) {
        if (!mbar_wait_hint(tempty + buf, bph ^ 1, &g_err, 52, a.wait_ns)) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * P::kAccCols;
        for (int kb = 0; kb < a.kblocks; ++kb) {
          if (!mbar_wait_hint(full + s, ph, &g_err, 53, a.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int nk = min(kBK / kStep, a.steps - kb * (kBK / kStep));
          const uint64_t ad = ad0 + (uint64_t)((s * kABytes) >> 4), bd = bd0 + (uint64_t)((s * P::kBBytes) >> 4);
#pragma unroll
          for (int k = 0; k < kBK / kStep; ++k)
            if (k < nk) mma_i8_pair(d, ad + 2 * k, bd + 2 * k, idesc_i8(256, BN), (kb != 0 || k != 0) ? 1u : 0u);
          commit_pair(empty + s);
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
        }
        if (ok) commit_pair(tfull + buf);
        if (++buf == P::kAcc) {
          buf = 0;
          bph ^= 1;
        }
      }
      // every MMA issued has finished before the TMEM is freed
      commit_pair(drain);
      mbar_wait_hint(drain, 0, nullptr, 0, a.wait_ns);
    }
  } else {
    // two warps per quadrant of TMEM lanes, each with half of the columns
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const uint32_t acc0 = tmem + ((uint32_t)(quad * 32) << 16) + half * kHalf;
    int buf = 0;
    uint32_t bph = 0;
    float* s_ws = reinterpret_cast<float*>(s_epi) + (warp - 2) * (2 * kHalf + kOutWords);   // [128] weight scales
    float* s_bias = s_ws + kHalf;                                                            // [128]
    uint32_t* s_out = reinterpret_cast<uint32_t*>(s_bias + kHalf);                           // [32 rows][17 words]
    pdl_wait_primary();                                // (the token scales)
    for (int tile = pair; tile < ntiles; tile += pairs) {
      int mb, nb;
      tile_at(a, tile, &mb, &nb);
      const int64_t m0 = (int64_t)mb * 256 + rank * 128 + quad * 32;
      const int64_t n0 = (int64_t)nb * BN + half * kHalf;
      const int cols = (int)max((int64_t)0, min((int64_t)kHalf, a.N - n0));
      const int rows = (int)max((int64_t)0, min((int64_t)32, a.M - m0));
      __syncwarp();                                    // (the last tile's scales have been used)
#pragma unroll
      for (int i = 0; i < (kHalf + 31) / 32; ++i) {
        const int col = i * 32 + lane;
        if (col >= kHalf) break;
        s_ws[col] = col < cols ? a.wscales[n0 + col] : 0.f;
        s_bias[col] = a.bias != nullptr && col < cols ? load_f(a.bias, a.bias_dtype, n0 + col) : 0.f;
      }
      const float xs = lane < rows ? a.xscales[m0 + lane] : 0.f;
      __syncwarp();
      const bool got = mbar_wait_hint(tfull + buf, bph, &g_err, 54, a.wait_ns);
      if (!__all_sync(0xffffffffu, got)) break;
      tc_fence_after();
      // A few columns at a time, by one short loop: a tile's whole epilogue unrolled is 16 KB of
      // instructions, which cost a small call 4 us to fetch.
      constexpr int CW = kHalf % 32 == 0 ? 32 : 16;
      const uint32_t acc = acc0 + buf * P::kAccCols;
      const bool words = (reinterpret_cast<uintptr_t>(a.out) & 3) == 0 && (a.out_stride & 1) == 0;
#pragma unroll 1
      for (int c = 0; c < kHalf; c += CW) {
        float f[CW];
        if constexpr (CW == 32) tmem_ld32(acc + c, f);
        else tmem_ld16(acc + c, f);
        if (c + CW >= kHalf) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_cluster(map_cta(smem_u32(tempty + buf), 0));
        }
        if (rows == 0 || c >= cols) continue;
#pragma unroll
        for (int i = 0; i < CW; i += 4) {
          const float4 ws = *reinterpret_cast<const float4*>(s_ws + c + i), bs = *reinterpret_cast<const float4*>(s_bias + c + i);
          f[i] = scaled(__float_as_int(f[i]), xs, ws.x, bs.x);
          f[i + 1] = scaled(__float_as_int(f[i + 1]), xs, ws.y, bs.y);
          f[i + 2] = scaled(__float_as_int(f[i + 2]), xs, ws.z, bs.z);
          f[i + 3] = scaled(__float_as_int(f[i + 3]), xs, ws.w, bs.w);
        }
        if (a.out_dtype == TS_F32) {
          float* out = reinterpret_cast<float*>(a.out) + m0 * a.out_stride + n0 + c;
          if (a.vec) {                                 // N is a multiple of 4
            float* row = out + lane * a.out_stride;
#pragma unroll
            for (int i = 0; i < CW; i += 4)
              if (lane < rows && c + i < cols) *reinterpret_cast<float4*>(row + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
            continue;
          }
          // 16 columns of the warp's rows at a time through shared memory, two
          // rows of them per store
#pragma unroll
          for (int h = 0; h < CW; h += 16) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 16; ++j) s_out[lane * 17 + j] = __float_as_uint(f[h + j]);
            __syncwarp();
            const int col = h + (lane & 15);
            for (int r = lane >> 4; r < rows; r += 2)
              if (c + col < cols) out[r * a.out_stride + col] = __uint_as_float(s_out[r * 17 + (lane & 15)]);
          }
          continue;
        }
        uint32_t v[CW / 2];
#pragma unroll
        for (int i = 0; i < CW / 2; ++i)
          v[i] = a.out_dtype == TS_BF16 ? paged::pack2<true>(f[2 * i], f[2 * i + 1]) : paged::pack2<false>(f[2 * i], f[2 * i + 1]);
        uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + m0 * a.out_stride + n0 + c;
        if (a.vec) {                                   // N is a multiple of 8
          uint16_t* row = out + lane * a.out_stride;
#pragma unroll
          for (int i = 0; i < CW / 8; ++i)
            if (lane < rows && c + i * 8 < cols)
              *reinterpret_cast<uint4*>(row + i * 8) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          continue;
        }
        // through shared memory: rows by words where they start on words, else by elements
        __syncwarp();
#pragma unroll
        for (int j = 0; j < CW / 2; ++j) s_out[lane * 17 + j] = v[j];
        __syncwarp();
        if (words) {
          constexpr int kPer = 64 / CW;                // rows of a store
          const int w = lane % (CW / 2), col = 2 * w;
          for (int r = lane / (CW / 2); r < rows; r += kPer) {
            const uint32_t x = s_out[r * 17 + w];
            uint16_t* dst = out + r * a.out_stride + col;
            if (c + col + 1 < cols) *reinterpret_cast<uint32_t*>(dst) = x;
            else if (c + col < cols) *dst = (uint16_t)x;
          }
        } else {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(s_out);
          constexpr int kPer = 32 / CW;                // rows of a store
          const int col = lane % CW;
          for (int r = lane / CW; r < rows; r += kPer)
            if (c + col < cols) out[r * a.out_stride + col] = h[r * 34 + col];
        }
      }
      if (++buf == P::kAcc) {
        buf = 0;
        bph ^= 1;
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
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P::kAcc * P::kAccCols) : "memory");
  }
}

// ---- host -------------------------------------------------------------------

struct Plan {
  int pair;         // CTA pairs on tiles of 256 tokens x this many weight rows, or 0
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
    auto k = int8_gemm_kernel<128, false>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(sm_count() / size * size));
    cfg.blockDim = dim3((unsigned)kThreads);
    cfg.dynamicSmemBytes = Shape<128>::kSmem;
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

// Cycles that a call takes, as measured (0.5 to 2 us of launch and first loads aside): a stage
// of a pair's tile what its bytes take into an SM at 60 a cycle, the change from tile to
// tile 500; a stage of a lone CTA's tile its bytes at 40 a cycle, or the weight's at DRAM's
// rate, 1400 for the results of each 32 tokens, 500 and 1200 per 32 tokens for the join of up to four
// pieces, 1500 and 600 for a cluster's. Both kinds of plan tried on 4 weights x 12 numbers of tokens from 1 to
// 4096: the one taken is within 5% of the best, but for 33 to 64 tokens, where the costs of a lone CTA's results are not
// told well (6144 x 4096 14.4 us, pairs of 96 rows 11.4; 14336 x 4096 18.1 us, lone CTAs 16.7; 4096 x 4096, 64 tokens 11.2,
// pairs of 64 rows 10.1). Up to 32 tokens a pair's tile of 256 is all but empty (1 x 14336
// x 4096: 23 us, a lone CTA's 13.6).
static Plan plan(int64_t M, int64_t N, int64_t K) {
  Plan p{};
  const int sms = std::max(2, sm_count()), pairs = sms / 2;
  p.kblocks = (int)((K + kBK - 1) / kBK);
  p.BT = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  p.wblocks = (int)((N + kBW - 1) / kBW);
  p.tblocks = (int)((M + p.BT - 1) / p.BT);
  const int64_t ntiles = (int64_t)p.wblocks * p.tblocks, units = ntiles * p.kblocks;
  const int rounds = (int)(std::min<int64_t>(M, p.BT) + 31) / 32;
  const double stream = (double)units * kABytes / 3300;   // the weight's bytes, at DRAM's bytes per cycle
  auto cost = [&](int64_t grid, int pieces) {
    const double own = (double)((units + grid - 1) / grid) * (kABytes + p.BT * kBK) / 40;
    return std::max(own, stream) + (pieces > 1 ? 500 + 1200.0 * rounds * ((pieces + 3) / 4) : 0) +
           (double)((ntiles + grid - 1) / grid) * rounds * 1400;
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
  if (M <= 32) return p;
  const int64_t mb = (M + 255) / 256;
  bool take = ntiles > (int64_t)paged::kCounters;
  for (int bn : {256, 224, 192, 160, 128, 96, 64}) {
    const int64_t nb = (N + bn - 1) / bn, tiles = mb * nb;
    const double c = (double)((tiles + pairs - 1) / pairs) * ((kABytes + bn * 64) / 60.0 * p.kblocks + 500) + 1500;
    if (take ? p.pair != 0 && c >= best : c >= best) continue;
    best = c;
    take = true;
    p.pair = bn;
    p.cluster = 0;
    p.tblocks = (int)mb;
    p.wblocks = (int)std::min<int64_t>(nb, INT32_MAX);
    p.ntiles = (int)std::min<int64_t>(tiles, INT32_MAX);
    p.grid = 2 * (int)std::min<int64_t>(tiles, pairs);
  }
  return p;
}

template <int BT, bool Q>
static int launch(const CUtensorMap& wm, const CUtensorMap& xm, const GemmArgs& a, int grid, int overlap, cudaStream_t st) {
  auto k = int8_gemm_kernel<BT, Q>;
  constexpr size_t smem = Shape<BT>::kSmem;
  static_assert(smem <= 227 * 1024, "shared memory");
  static thread_local int configured_dev = -1;
  int dev = 0;
  TS_CUDA_TRY(cudaGetDevice(&dev));
  if (configured_dev != dev) {
    TS_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    configured_dev = dev;
  }
  TS_CUDA_TRY(launch_after(k, grid, kThreads + (Q ? kQuantWarps * 32 : 0), smem, st, overlap, a.cluster, wm, xm, a));
  TS_LAUNCH_CHECK();
  return TS_OK;
}

template <int BN>
static int launch_pair(const CUtensorMap& am, const CUtensorMap& bm, const PairArgs& a, int grid, int overlap, cudaStream_t st) {
  constexpr size_t smem = Pair<BN>::kSmem;
  static_assert(smem <= 227 * 1024, "shared memory");
  auto k = int8_pair_kernel<BN>;
  static thread_local int configured_dev = -1;
  int dev = 0;
  TS_CUDA_TRY(cudaGetDevice(&dev));
  if (configured_dev != dev) {
    TS_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    configured_dev = dev;
  }
  TS_CUDA_TRY(launch_after(k, grid, kPairThreads, smem, st, overlap, 0, am, bm, a));
  TS_LAUNCH_CHECK();
  return TS_OK;
}

// Bytes of a plan's workspace: counters, then partial sums.
static size_t plan_bytes(const Plan& p) {
  return paged::kCounterBytes + (!p.pair && !p.cluster ? (size_t)p.grid * 2 * kBW * p.BT * 4 : 0);
}

// Tokens that the product quantises itself.
struct Tokens {
  const void* x;
  int dtype;
  int64_t stride;
};

static int matmul(const Plan& p, const ts_int8_tensor* x, const ts_int8_tensor* w, const void* bias, int bias_dtype, void* out,
                  int out_dtype, int64_t out_row_stride, void* workspace, size_t workspace_bytes, int overlap, const Tokens* own,
                  void* stream) {
  TS_UNSUPPORTED(out_dtype == TS_F16 || out_dtype == TS_BF16 || out_dtype == TS_F32, "unknown output type %d", out_dtype);
  TS_UNSUPPORTED(!bias || bias_dtype == TS_F16 || bias_dtype == TS_BF16 || bias_dtype == TS_F32, "unknown bias type %d",
                 bias_dtype);
  TS_REQUIRE(out && is_aligned(out, out_dtype == TS_F32 ? 4 : 2), "out must be aligned to its elements");
  const size_t need = plan_bytes(p);
  if (!p.pair && (workspace == nullptr || workspace_bytes < need)) {
    set_error("workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return TS_ERR_WORKSPACE;
  }
  TS_REQUIRE(is_aligned(workspace, 16), "workspace must be 16-byte aligned");
  TS_UNSUPPORTED(p.pair || p.ntiles <= (int)paged::kCounters, "too many output features in one call");
  TS_UNSUPPORTED(p.ntiles < INT32_MAX, "too many outputs in one call");
  const int steps = (int)((w->cols + kStep - 1) / kStep);
  const int stall = take_test_stall() ? 1 : 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto map = [&](CUtensorMap* m, const ts_int8_tensor* t, uint32_t rows) {
    // (columns behind the last come as zeros, whatever the padding holds)
    return encode_tmap_2d(m, t->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, (uint64_t)t->cols, (uint64_t)t->rows,
                          (uint64_t)t->row_stride, kBK, rows, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  CUtensorMap wm, xm;
  int rc = map(&wm, w, p.pair ? p.pair / 2 : kBW);
  if (own) xm = wm;                                    // (not used)
  else if (rc == TS_OK) rc = map(&xm, x, p.pair ? 128 : p.BT);
  if (rc != TS_OK) return rc;
  if (p.pair) {
    PairArgs a;
    a.wscales = w->scales;
    a.xscales = x->scales;
    a.M = x->rows;
    a.N = w->rows;
    a.mblocks = p.tblocks;
    a.nblocks = p.wblocks;
    a.kblocks = p.kblocks;
    a.group = (int)std::max<int64_t>(1, std::min<int64_t>(a.mblocks, (32 << 20) / (256 * w->cols)));
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
    switch (p.pair) {
      case 64: return launch_pair<64>(xm, wm, a, p.grid, overlap, st);
      case 96: return launch_pair<96>(xm, wm, a, p.grid, overlap, st);
      case 128: return launch_pair<128>(xm, wm, a, p.grid, overlap, st);
      case 160: return launch_pair<160>(xm, wm, a, p.grid, overlap, st);
      case 192: return launch_pair<192>(xm, wm, a, p.grid, overlap, st);
      case 224: return launch_pair<224>(xm, wm, a, p.grid, overlap, st);
      default: return launch_pair<256>(xm, wm, a, p.grid, overlap, st);
    }
  }
  GemmArgs a;
  a.wscales = w->scales;
  a.xscales = x->scales;
  a.M = x->rows;
  a.N = w->rows;
  a.wblocks = p.wblocks;
  a.tblocks = p.tblocks;
  a.kblocks = p.kblocks;
  a.steps = steps;
  a.bias = bias;
  a.bias_dtype = bias_dtype;
  a.out = out;
  a.out_dtype = out_dtype;
  a.out_stride = out_row_stride;
  a.counters = reinterpret_cast<int*>(workspace);
  a.partials = reinterpret_cast<int*>(reinterpret_cast<char*>(workspace) + paged::kCounterBytes);
  a.wait_ns = wait_limit_ns();
  a.stall = stall;
  a.cluster = p.cluster;
  const int wide = out_dtype == TS_F32 ? 16 : 8;       // bytes of four values
  a.out_vec = is_aligned(out, wide) && out_row_stride % 4 == 0;
  a.x = own ? own->x : nullptr;
  a.x_dtype = own ? own->dtype : 0;
  a.x_stride = own ? own->stride : 0;
  a.x_aligned = own && is_aligned(own->x, 16) && own->stride * (own->dtype == TS_F32 ? 4 : 2) % 16 == 0;
  a.K = w->cols;
  static_assert(kOwnTokens <= 16, "tokens of the kernel that quantises them");
  if (own) return launch<16, true>(wm, xm, a, p.grid, 0, st);
  switch (p.BT) {
    case 16: return launch<16, false>(wm, xm, a, p.grid, overlap, st);
    case 32: return launch<32, false>(wm, xm, a, p.grid, overlap, st);
    case 64: return launch<64, false>(wm, xm, a, p.grid, overlap, st);
    default: return launch<128, false>(wm, xm, a, p.grid, overlap, st);
  }
}

}  // namespace int8
}  // namespace ts

using namespace ts;
using namespace ts::int8;

extern "C" size_t ts_int8_matmul_workspace_size(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return paged::kCounterBytes;
  return plan_bytes(plan(M, N, K));
}

extern "C" int ts_int8_matmul(const ts_int8_tensor* a, const ts_int8_tensor* b, const void* bias, int bias_dtype, void* out,
                              int out_dtype, int64_t out_row_stride, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_tensor(a, "ts_int8_matmul a");
  if (rc != TS_OK) return rc;
  rc = check_tensor(b, "ts_int8_matmul b");
  if (rc != TS_OK) return rc;
  TS_REQUIRE(a->cols == b->cols, "a has %lld columns, b %lld", (long long)a->cols, (long long)b->cols);
  if (a->rows == 0 || b->rows == 0) return TS_OK;
  return matmul(plan(a->rows, b->rows, b->cols), a, b, bias, bias_dtype, out, out_dtype, out_row_stride, workspace,
                workspace_bytes, 0, nullptr, stream);
}

extern "C" int ts_int8_status(int clear, void* stream) {
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int v = 0;
  TS_CUDA_TRY(cudaMemcpyFromSymbolAsync(&v, g_err, sizeof(int), 0, cudaMemcpyDeviceToHost, st));
  TS_CUDA_TRY(cudaStreamSynchronize(st));
  if (v == 0) return TS_OK;
  if (clear) {
    const int zero = 0;
    TS_CUDA_TRY(cudaMemcpyToSymbolAsync(g_err, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st));
    TS_CUDA_TRY(cudaStreamSynchronize(st));
  }
  set_error("a bounded wait in the int8 product ran out (code %d); the outputs of the calls since the last "
            "status check are not valid", v);
  return TS_ERR_TIMEOUT;
}

// ---- quantised activations and the product in one call ----------------------

static size_t linear_act_bytes(int64_t M, int64_t K) {
  return align_up((size_t)M * (size_t)padded_cols(K), 256) + align_up((size_t)M * 4, 256);
}

extern "C" size_t ts_int8_linear_workspace_size(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return paged::kCounterBytes;
  return align_up(ts_int8_matmul_workspace_size(M, N, K), 256) + linear_act_bytes(M, K);
}

extern "C" int ts_int8_linear(const void* x, int x_dtype, int64_t M, int64_t x_row_stride, const ts_int8_tensor* w,
                              const void* bias, int bias_dtype, void* out, int out_dtype, int64_t out_row_stride,
                              void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_tensor(w, "ts_int8_linear w");
  if (rc != TS_OK) return rc;
  TS_REQUIRE(M >= 0, "bad shape");
  if (M == 0 || w->rows == 0) return TS_OK;
  const Plan p = plan(M, w->rows, w->cols);
  // the activations' codes and scales lie behind the product's scratch
  const size_t at = align_up(plan_bytes(p), 256), need = at + linear_act_bytes(M, w->cols);
  if (workspace == nullptr || workspace_bytes < need) {
    set_error("workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return TS_ERR_WORKSPACE;
  }
  TS_REQUIRE(is_aligned(workspace, 16), "workspace must be 16-byte aligned");
  ts_int8_tensor t{};
  t.codes = reinterpret_cast<int8_t*>(workspace) + at;
  t.row_stride = padded_cols(w->cols);
  t.scales = reinterpret_cast<float*>(t.codes + align_up((size_t)M * (size_t)t.row_stride, 256));
  t.rows = M;
  t.cols = w->cols;
  if (M <= kOwnTokens && M * w->cols <= kOwnElements) {
    TS_UNSUPPORTED(x_dtype == TS_F16 || x_dtype == TS_BF16 || x_dtype == TS_F32, "unknown element type %d", x_dtype);
    TS_REQUIRE(x && is_aligned(x, x_dtype == TS_F32 ? 4 : 2), "x must be aligned to its elements");
    const Tokens own = {x, x_dtype, x_row_stride};
    return matmul(p, &t, w, bias, bias_dtype, out, out_dtype, out_row_stride, workspace, at, 0, &own, stream);
  }
  rc = ts_int8_quantize(x, x_dtype, x_row_stride, &t, stream);
  if (rc != TS_OK) return rc;
  return matmul(p, &t, w, bias, bias_dtype, out, out_dtype, out_row_stride, workspace, at, 1, nullptr, stream);
}
