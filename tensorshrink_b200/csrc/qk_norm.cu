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
// rotation once for all of them; few tokens are spread over more warps instead. 8191
// tokens of 64 query heads over 8 of 128 columns, stored too: 69 us, 5.4 TB/s (with the
// position loaded where it is needed, and one operation at a time: 85 us; two heads a
// lane: 88 us). One token of 32 heads over 8: 3.0 us in a graph.
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
  float eps, inv_dim;
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

// Eight values from column j on.
__device__ __forceinline__ void load8(const void* w, int dtype, int j, Two (&f)[4]) {
  if (dtype == TS_F32) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(w) + j));
    const float4 b = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(w) + j) + 1);
    f[0] = two(a.x, a.y);
    f[1] = two(a.z, a.w);
    f[2] = two(b.x, b.y);
    f[3] = two(b.z, b.w);
  } else {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(w) + j));
    const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = dtype == TS_BF16 ? unpack2<true>(q[i]) : unpack2<false>(q[i]);
      f[i] = two(v.x, v.y);
    }
  }
}

// L: lanes of a head. U: heads of a lane.
template <bool BF, int L, int U>
__global__ void __launch_bounds__(256, 2) qk_norm_rope_kernel(const NormArgs a) {
  constexpr int kPer = 32 / L;                       // heads of a warp at a time
  const int lane = threadIdx.x & 31, lh = lane / L, lc = lane % L;
  const int D = a.head_dim, half = D / 2, j = lc * 8;
  const bool on = lc < D / 16;
  const int groups = (a.heads + kPer * U - 1) / (kPer * U);
  // this warp's items (a token, a group of its heads), one stride apart
  const int64_t first = blockIdx.x * (int64_t)8 + (threadIdx.x >> 5), stride = (int64_t)gridDim.x * 8;
  const int64_t t_step = stride / groups;
  const int g_step = (int)(stride - t_step * groups);
  int64_t t = first / groups;
  int g = (int)(first - t * groups);
  const bool turn = a.cos_t != nullptr;
  // (the next item's position and slot are loaded an item ahead: rotation and store hang on them)
  auto position = [&](int64_t t) { return a.positions != nullptr && t < a.tokens ? a.positions[t] : 0; };
  auto place = [&](int64_t t) { return a.slots != nullptr && t < a.tokens ? a.slots[t] : -1; };
  int64_t pos = position(t), slot = place(t);
  while (t < a.tokens) {
    const int head0 = g * (kPer * U) + lh;
    const int64_t now = t;
    t += t_step;
    g += g_step;
    if (g >= groups) {
      g -= groups;
      ++t;
    }
    const int64_t pos_next = position(t), slot_next = place(t);
    const uint16_t* row = a.x + now * a.x_stride + head0 * D + j;
    uint4 lo[U], hi[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
      if (on && head0 + u * kPer < a.heads) {
        lo[u] = *reinterpret_cast<const uint4*>(row + u * kPer * D);
        hi[u] = *reinterpret_cast<const uint4*>(row + u * kPer * D + half);
      }
    }
    const bool ok = !turn || (pos >= 0 && pos < a.rope_rows);
    Two cs[4], sn[4], ns[4];                           // cosines, sines and their negatives
    if (turn && ok && on) {
      load8(a.cos_t + pos * half, TS_F32, j, cs);
      load8(a.sin_t + pos * half, TS_F32, j, sn);
#pragma unroll
      for (int e = 0; e < 4; ++e) ns[e] = sn[e] ^ 0x8000000080000000ull;
    }
    // the slot in the pages
    int page = -1, off = 0;
    if (slot >= 0 && ok) {
      const int64_t p = a.page_shift >= 0 ? slot >> a.page_shift : slot / a.c.page_size;
      if (p < a.c.num_pages) {
        page = (int)p;
        off = (int)(slot - p * a.c.page_size);
      }
    }
    uint16_t* out = a.out + now * a.out_stride + head0 * D + j;
    const void* have = nullptr;                        // whose weights are in w
    Two w[8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = head0 + u * kPer;
      const bool is_q = h < a.n_q, is_k = !is_q && h < a.n_q + a.n_kv;
      const void* weight = is_q ? a.qw : is_k ? a.kw : nullptr;
      uint32_t* wl = reinterpret_cast<uint32_t*>(&lo[u]);
      uint32_t* wh = reinterpret_cast<uint32_t*>(&hi[u]);
      Two x[8];                                        // columns j .. j + 7, then their partners
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 p = unpack2<BF>(wl[e]), q = unpack2<BF>(wh[e]);
        x[e] = two(p.x, p.y);
        x[4 + e] = two(q.x, q.y);
      }
      Two squares = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) squares = fma2(x[e], x[e], squares);
      float sum = both(squares).x + both(squares).y;
#pragma unroll
      for (int s = L / 2; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
      if (!on || h >= a.heads) continue;
      if (is_q || is_k) {
        if (weight != nullptr) {
          if (weight != have) {
            load8(weight, a.w_dtype, j, *reinterpret_cast<Two(*)[4]>(w));
            load8(weight, a.w_dtype, j + half, *reinterpret_cast<Two(*)[4]>(w + 4));
            have = weight;
          }
          const float r = rsqrtf(sum * a.inv_dim + a.eps);
          const Two rr = two(r, r);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = mul2(mul2(x[e], rr), w[e]);
        }
        if (turn && ok) {
          // (products and sums rounded one by one, as `rotate` does)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const Two y = add2(mul2_rn(x[e], cs[e]), mul2_rn(x[4 + e], ns[e]));
            x[4 + e] = add2(mul2_rn(x[e], sn[e]), mul2_rn(x[4 + e], cs[e]));
            x[e] = y;
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          wl[e] = ok ? pack2<BF>(both(x[e]).x, both(x[e]).y) : 0;
          wh[e] = ok ? pack2<BF>(both(x[4 + e]).x, both(x[4 + e]).y) : 0;
        }
      } else if (!ok) {
        lo[u] = hi[u] = make_uint4(0, 0, 0, 0);
      }
      if (is_q || is_k || a.copy_v) {
        *reinterpret_cast<uint4*>(out + u * kPer * D) = lo[u];
        *reinterpret_cast<uint4*>(out + u * kPer * D + half) = hi[u];
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
    pos = pos_next;
    slot = slot_next;
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
  a.inv_dim = 1.f / (float)head_dim;
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
