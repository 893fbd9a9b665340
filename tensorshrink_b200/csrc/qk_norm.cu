// Norms of queries and keys for each head, with the rotation in the same pass and,
// for a paged cache, the store of keys and values.
//
//   y = x rsqrt(mean x^2 + eps) w,   (y1 c - y2 s, y1 s + y2 c)
//
// in fp32, rounded once. Bound by DRAM traffic: every element is read and written once. A
// lane holds 8 columns of a head's first half and their partners of the second,
// so that the rotation needs no exchange; D / 16 lanes of a power of two share a
// head and its sum of squares. A warp takes neighbouring heads of one token, up to
// kUnroll of them per lane with all loads in flight, and reads the token's
// rotation once for all of them; few tokens are spread over more warps instead.
#include <algorithm>

#include "paged.cuh"

namespace ts {
namespace paged {

struct NormArgs {
  const uint16_t* x;
  int64_t x_stride, tokens;
  int n_q, n_kv, head_dim;
  int heads;             // of a token that are processed: queries, keys and, where they move, values
  const void* qw;
  const void* kw;
  int w_dtype;
  float eps;
  const int64_t* positions;
  const float* cos_t;
  const float* sin_t;
  int64_t rope_rows;
  uint16_t* out;         // or NULL where only the store is left (never for queries)
  int64_t out_stride;
  int copy_v;            // values go to out
  Cache c;
  const int64_t* slots;  // or NULL
  int page_shift;
};

// Eight weights from column j on.
__device__ __forceinline__ void load_w(const void* w, int dtype, int j, float (&f)[8]) {
  if (dtype == TS_F32) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(w) + j));
    const float4 b = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(w) + j) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(w) + j));
    const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = dtype == TS_BF16 ? unpack2<true>(q[i]) : unpack2<false>(q[i]);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}

// L: lanes of a head. U: heads of a lane.
template <bool BF, int L, int U>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const NormArgs a) {
  constexpr int kPer = 32 / L;                       // heads of a warp at a time
  const int lane = threadIdx.x & 31, lh = lane / L, lc = lane % L;
  const int D = a.head_dim, half = D / 2, j = lc * 8;
  const bool on = lc < D / 16;
  const int groups = (a.heads + kPer * U - 1) / (kPer * U);
  const int64_t items = a.tokens * groups;
  for (int64_t it = blockIdx.x * (int64_t)8 + (threadIdx.x >> 5); it < items; it += (int64_t)gridDim.x * 8) {
    const int64_t t = it / groups;
    const int head0 = (int)(it - t * groups) * (kPer * U) + lh;
    const uint16_t* row = a.x + t * a.x_stride;
    uint4 lo[U], hi[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = head0 + u * kPer;
      lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
      if (on && h < a.heads) {
        lo[u] = *reinterpret_cast<const uint4*>(row + h * D + j);
        hi[u] = *reinterpret_cast<const uint4*>(row + h * D + j + half);
      }
    }
    const bool turn = a.cos_t != nullptr;
    const int64_t pos = a.positions != nullptr ? a.positions[t] : 0;
    const bool ok = !turn || (pos >= 0 && pos < a.rope_rows);
    float cs[8], sn[8];
    if (turn && ok && on) {
      const float* cp = a.cos_t + pos * half + j;
      const float* sp = a.sin_t + pos * half + j;
      load_w(cp, TS_F32, 0, cs);
      load_w(sp, TS_F32, 0, sn);
    }
    // the slot in the pages
    int page = -1, off = 0;
    if (a.slots != nullptr) {
      const int64_t s = a.slots[t];
      if (s >= 0 && ok) {
        const int64_t p = a.page_shift >= 0 ? s >> a.page_shift : s / a.c.page_size;
        if (p < a.c.num_pages) {
          page = (int)p;
          off = (int)(s - p * a.c.page_size);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = head0 + u * kPer;
      const bool is_q = h < a.n_q, is_k = !is_q && h < a.n_q + a.n_kv;
      const void* w = is_q ? a.qw : is_k ? a.kw : nullptr;
      uint32_t* wl = reinterpret_cast<uint32_t*>(&lo[u]);
      uint32_t* wh = reinterpret_cast<uint32_t*>(&hi[u]);
      float sum = 0.f;
      float x[16];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 p = unpack2<BF>(wl[e]), q = unpack2<BF>(wh[e]);
        x[2 * e] = p.x; x[2 * e + 1] = p.y;
        x[8 + 2 * e] = q.x; x[8 + 2 * e + 1] = q.y;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
      for (int s = L / 2; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
      if (!on || h >= a.heads) continue;
      if (is_q || is_k) {
        if (w != nullptr) {
          const float r = rsqrtf(sum / (float)D + a.eps);
          float w1[8], w2[8];
          load_w(w, a.w_dtype, j, w1);
          load_w(w, a.w_dtype, j + half, w2);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = x[e] * r * w1[e];
            x[8 + e] = x[8 + e] * r * w2[e];
          }
        }
        if (turn) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 y = ok ? rotate(x[e], x[8 + e], cs[e], sn[e]) : make_float2(0.f, 0.f);
            x[e] = y.x;
            x[8 + e] = y.y;
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          wl[e] = pack2<BF>(x[2 * e], x[2 * e + 1]);
          wh[e] = pack2<BF>(x[8 + 2 * e], x[8 + 2 * e + 1]);
        }
      } else if (!ok) {
        lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
      }
      if (is_q || is_k || a.copy_v) {
        uint16_t* o = a.out + t * a.out_stride + h * D + j;
        *reinterpret_cast<uint4*>(o) = lo[u];
        *reinterpret_cast<uint4*>(o + half) = hi[u];
      }
      if (page >= 0 && !is_q) {
        const int kh = is_k ? h - a.n_q : h - a.n_q - a.n_kv;
        uint16_t* o = reinterpret_cast<uint16_t*>(is_k ? a.c.k : a.c.v) + row_at(a.c, page, kh, off) + j;
        *reinterpret_cast<uint4*>(o) = lo[u];
        *reinterpret_cast<uint4*>(o + half) = hi[u];
        if (is_k && lc == 0) {
          const int64_t sa = stat_at(a.c, page, kh, off);
          if (a.c.scores != nullptr) a.c.scores[sa] = 0.f;
          if (a.c.slot_pos != nullptr) a.c.slot_pos[sa] = (int32_t)pos;
        }
      }
    }
  }
}

template <bool BF, int L>
static void launch_norm(const NormArgs& a, cudaStream_t st) {
  constexpr int kPer = 32 / L, kUnroll = 4;
  const int64_t ctas = (int64_t)sm_count() * 8;
  auto grid = [&](int u) {
    const int64_t items = a.tokens * ((a.heads + kPer * u - 1) / (kPer * u));
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + 7) / 8, ctas));
  };
  // several heads a lane where there are warps enough without them
  if (a.tokens * a.heads >= (int64_t)sm_count() * 8 * kPer * kUnroll) qk_norm_rope_kernel<BF, L, kUnroll><<<grid(kUnroll), 256, 0, st>>>(a);
  else qk_norm_rope_kernel<BF, L, 1><<<grid(1), 256, 0, st>>>(a);
}

template <bool BF>
static void launch_norm(const NormArgs& a, cudaStream_t st) {
  const int lanes = a.head_dim / 16;
  if (lanes <= 1) launch_norm<BF, 1>(a, st);
  else if (lanes <= 2) launch_norm<BF, 2>(a, st);
  else if (lanes <= 4) launch_norm<BF, 4>(a, st);
  else if (lanes <= 8) launch_norm<BF, 8>(a, st);
  else launch_norm<BF, 16>(a, st);
}

}  // namespace paged
}  // namespace ts

using namespace ts;
using namespace ts::paged;

extern "C" int ts_qk_norm_rope(const void* x, int dtype, int64_t x_row_stride, int64_t tokens, int n_q, int n_kv, int head_dim,
                               const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                               const int64_t* positions, const float* rope_cos, const float* rope_sin, int64_t rope_rows,
                               void* out, int64_t out_row_stride, const ts_paged_cache* cache, const int64_t* slots,
                               void* stream) {
  TS_UNSUPPORTED(dtype == TS_F16 || dtype == TS_BF16, "x must be fp16 or bf16");
  TS_REQUIRE(tokens >= 0 && n_q >= 0 && n_kv >= 0 && n_q + n_kv > 0, "bad sizes");
  TS_UNSUPPORTED(head_dim % 16 == 0 && head_dim >= 16 && head_dim <= 256, "head_dim must be a multiple of 16, <= 256");
  TS_UNSUPPORTED(((int64_t)n_q + 2 * (int64_t)n_kv) * head_dim < (int64_t)1 << 31, "too many heads");
  TS_UNSUPPORTED((q_weight == nullptr && k_weight == nullptr) || weight_dtype == TS_F32 || weight_dtype == dtype,
                 "weights must be fp32 or of x's type");
  TS_REQUIRE((rope_cos == nullptr) == (rope_sin == nullptr), "rope_cos and rope_sin come both or neither");
  TS_REQUIRE(eps >= 0.f && eps < INFINITY, "eps must not be negative");
  TS_REQUIRE((cache == nullptr) == (slots == nullptr), "a cache and slots come both or neither");
  NormArgs a{};
  if (cache != nullptr) {
    const int rc = make_cache(cache, &a.c);
    if (rc != TS_OK) return rc;
    TS_REQUIRE(cache->dtype == dtype && cache->n_kv == n_kv && cache->head_dim == head_dim, "the cache does not fit x");
    TS_REQUIRE(cache->slot_pos == nullptr || positions != nullptr, "positions are needed for slot_pos");
    a.page_shift = log2_of(cache->page_size);
  }
  if (tokens == 0) return TS_OK;
  TS_REQUIRE(x && out, "NULL pointer");
  TS_REQUIRE(positions != nullptr || rope_cos == nullptr, "positions are needed for the rotation");
  TS_REQUIRE(is_aligned(x, 16) && is_aligned(out, 16) && x_row_stride % 8 == 0 && out_row_stride % 8 == 0,
             "rows of x and out must be 16-byte aligned");
  TS_REQUIRE(is_aligned(q_weight, 16) && is_aligned(k_weight, 16), "weights must be 16-byte aligned");
  TS_REQUIRE(is_aligned(rope_cos, 16) && is_aligned(rope_sin, 16), "rotary tables must be 16-byte aligned");
  a.x = reinterpret_cast<const uint16_t*>(x);
  a.x_stride = x_row_stride;
  a.tokens = tokens;
  a.n_q = n_q;
  a.n_kv = n_kv;
  a.head_dim = head_dim;
  a.qw = q_weight;
  a.kw = k_weight;
  a.w_dtype = weight_dtype;
  a.eps = eps;
  a.positions = positions;
  a.cos_t = rope_cos;
  a.sin_t = rope_sin;
  a.rope_rows = rope_rows;
  a.out = reinterpret_cast<uint16_t*>(out);
  a.out_stride = out_row_stride;
  // values in place stay where they are, unless a token may have to become zeros
  const bool in_place = x == out && x_row_stride == out_row_stride;
  a.copy_v = !in_place || rope_cos != nullptr;
  a.heads = n_q + n_kv + (!in_place || rope_cos != nullptr || slots != nullptr ? n_kv : 0);
  a.slots = slots;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == TS_BF16) launch_norm<true>(a, st);
  else launch_norm<false>(a, st);
  TS_LAUNCH_CHECK();
  return TS_OK;
}
