// Storing tokens in a paged cache of 8 bits, and its values.
//
// A warp takes one block of slots of one kv head, of k or of v: the new tokens that fall
// into it are loaded (16 bytes a lane, eight loads in flight), their largest
// magnitude gives the scale the block needs, and the codes are made from the registers that
// the tokens came into; rows behind the first eight loads of a lane (blocks of more
// than 16 rows of 128 columns) are read a second time, from L1 or L2. A block that
// holds earlier tokens keeps its scale where that is large enough. Where it is not, the
// scale grows by a quarter at least and the earlier codes are rounded anew. An int8 code is
// then off by 1/2 (1 + 0.8 + 0.64 + ...) < 2.5 steps at most however often its block's scale
// grows, where growth to what is needed would let the half steps of 15 tokens add up. An e4m3
// code's step shrinks with the code: m growths leave a value within (1 + 2^-4)^(m + 1) - 1 of itself (of
// 15 growths in a row, chosen to make it worst, 105%), which is at most 15% of the block's largest.
// Bound by DRAM traffic: the tokens are read once, codes of half the size written. 30000 packed
// tokens of 16 sequences, 8 heads of 128 columns, bf16 to e4m3: 38.5 us, 4.9 TB/s; the
// values of the pages that they fill 32 us, 5.9 TB/s; one token of 64 sequences 3.8 us.
#include <algorithm>

#include "paged8.cuh"

namespace ts {
namespace paged8 {

constexpr int kHold = 8;           // 16-byte loads of a lane that stay in registers

using paged::pack2;
using paged::unpack2;

// Eight neighbouring elements of a row of k or v; of k with tables, rotated and
// rounded to the type.
template <bool BF, bool ROPE>
__device__ __forceinline__ uint4 load_row(const uint16_t* row, int cc, int chunks, const float* cs, const float* sn) {
  uint4 w = *reinterpret_cast<const uint4*>(row + cc * 8);
  if (ROPE && cs != nullptr) {
    const int half = chunks / 2;
    const bool hi = cc >= half;
    const int j = (hi ? cc - half : cc) * 8;
    const uint4 p = *reinterpret_cast<const uint4*>(row + (hi ? cc - half : cc + half) * 8);
    uint32_t* ww = reinterpret_cast<uint32_t*>(&w);
    const uint32_t* pw = reinterpret_cast<const uint32_t*>(&p);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 x = unpack2<BF>(hi ? pw[e] : ww[e]), y = unpack2<BF>(hi ? ww[e] : pw[e]);
      const float2 r0 = paged::rotate(x.x, y.x, cs[j + 2 * e], sn[j + 2 * e]);
      const float2 r1 = paged::rotate(x.y, y.y, cs[j + 2 * e + 1], sn[j + 2 * e + 1]);
      ww[e] = hi ? pack2<BF>(r0.y, r1.y) : pack2<BF>(r0.x, r1.x);
    }
  }
  return w;
}

__device__ __forceinline__ uint32_t top_bits(const uint4& w) {
  const uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu), __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu));
  return max(m & 0xFFFFu, m >> 16);
}

template <bool BF, bool E4M3>
__device__ __forceinline__ uint2 codes_of(const uint4& w, float r) {
  const Two rr = two(r, r);
  auto pair = [&](uint32_t x) {
    const float2 f = unpack2<BF>(x);
    return mul2_rn(two(f.x, f.y), rr);
  };
  return make_uint2(encode4<E4M3>(pair(w.x), pair(w.y)), encode4<E4M3>(pair(w.z), pair(w.w)));
}

template <bool BF, bool E4M3, bool ROPE>
__global__ void __launch_bounds__(256, ROPE ? 2 : 4) paged8_append_kernel(const AppendArgs a) {
  const Cache& c = a.c;
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, b = blockIdx.y, len = c.seq_lens[b];
  int64_t base = 0, count = a.tokens;
  if (a.offsets != nullptr) {
    base = max(0, a.offsets[b]);
    count = min((int64_t)a.offsets[b + 1], a.tokens) - base;
  }
  if (a.n_new != nullptr) count = min(count, (int64_t)a.n_new[b]);
  const int64_t capacity = (int64_t)c.max_pages * c.page_size;
  if (len < 0 || len >= capacity || count <= 0) return;
  const int tokens = (int)min(count, capacity - len);  // those that have a slot
  const int64_t first = a.first != nullptr ? a.first[b] : len;
  const int chunks = c.head_dim / 8, per = 32 / chunks;         // rows of a step
  const int rl = lane / chunks, cc = lane - rl * chunks;        // this lane's row of a step and its chunk
  const bool on = rl < per;
  const int bs = c.block, blk0 = len / bs, blocks = (len + tokens - 1) / bs - blk0 + 1;
  const int items = blocks * c.n_kv * 2;
  // neighbouring warps take neighbouring heads of the same tokens
  for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < items; i += gridDim.x * 8) {
    const int hv = i % (c.n_kv * 2), h = hv % c.n_kv, is_v = hv / c.n_kv;
    const int slot0 = (blk0 + i / (c.n_kv * 2)) * bs;           // of the block
    const int page = c.table[b * c.table_stride + slot0 / c.page_size];
    const int off0 = slot0 % c.page_size;
    const int r0 = max(0, len - slot0), r1 = min(bs, len + tokens - slot0);   // the rows that get tokens
    const uint16_t* src = is_v ? a.v + h * a.vh : a.k + h * a.kh;
    const int64_t step = is_v ? a.vt : a.kt;
    const uint16_t* tok0 = src + (a.offsets != nullptr ? base * step : b * (is_v ? a.vb : a.kb)) + (int64_t)(slot0 - len) * step;
    const bool turn = ROPE && !is_v;
    const int64_t pos0 = first + (slot0 - len);
    // (a key whose position has no rotary row is dropped, and its value with it)
    int lo = r0, hi = on ? r1 : 0;                              // the rows that this lane may take
    if (ROPE) {
      lo = (int)max((int64_t)lo, min(-pos0, (int64_t)bs));
      hi = (int)min((int64_t)hi, max(a.rope_rows - pos0, (int64_t)0));
    }
    auto has = [&](int r) { return r < hi && (!ROPE || r >= lo); };
    auto load = [&](const uint16_t* row, int r) {
      const int64_t p = (pos0 + r) * (c.head_dim / 2);
      return load_row<BF, ROPE>(row, cc, chunks, turn ? a.cos_t + p : nullptr, turn ? a.sin_t + p : nullptr);
    };
    const uint16_t* row0 = tok0 + (r0 + rl) * step;             // of this lane's first row
    const int64_t row_step = per * step;
    uint4 w[kHold];
    uint32_t top = 0;
    bool any = false;
#pragma unroll
    for (int s = 0; s < kHold; ++s) {
      const int r = r0 + s * per + rl;
      w[s] = make_uint4(0, 0, 0, 0);
      if (has(r)) {
        w[s] = load(row0 + s * row_step, r);
        any = true;
      }
    }
    // (the tokens are on their way while the page is looked up)
    if ((unsigned)page >= (unsigned)c.num_pages) continue;
    uint8_t* out = (is_v ? c.v : c.k) + row_at(c, page, h, off0) + cc * 8;
    float* sp = (is_v ? c.v_scales : c.k_scales) + scale_at(c, page, h, off0 / bs);
    const float old = r0 > 0 ? *sp : 0.f;
#pragma unroll
    for (int s = 0; s < kHold; ++s) top = max(top, top_bits(w[s]));
    for (int r = r0 + kHold * per + rl; r < r1; r += per)
      if (has(r)) {
        top = max(top, top_bits(load(tok0 + r * step, r)));
        any = true;
      }
    if (!__any_sync(0xffffffffu, any)) continue;
    top = __reduce_max_sync(0xffffffffu, top);
    // the scale
    const bool finite = top < (BF ? 0x7F80u : 0x7C00u);
    float scale = __uint_as_float(0x7FC00000u);
    if (finite) {
      scale = scale_of<E4M3>(unpack2<BF>(top).x);
      if (r0 > 0) {
        if (scale > fabsf(old)) {
          scale = fmaxf(scale, __fmul_rn(1.25f, fabsf(old)));
          // the earlier tokens' codes, rounded anew
          const float ratio = __fdiv_rn(old, scale);
          for (int r = rl; r < r0; r += per)
            if (on) {
              uint2* p = reinterpret_cast<uint2*>(out + r * c.token_stride);
              const uint2 q = *p;
              const Two rr = two(ratio, ratio);
              float x[4], y[4];
              decode4<E4M3>(q.x, x);
              decode4<E4M3>(q.y, y);
              *p = make_uint2(encode4<E4M3>(mul2_rn(two(x[0], x[1]), rr), mul2_rn(two(x[2], x[3]), rr)),
                              encode4<E4M3>(mul2_rn(two(y[0], y[1]), rr), mul2_rn(two(y[2], y[3]), rr)));
            }
        } else {
          scale = old;                                 // (a NaN stays)
        }
      }
    }
    if (lane == 0) *sp = scale;
    const bool number = scale == scale;
    const float r = number ? __frcp_rn(scale) : 0.f;
    auto put = [&](uint8_t* row, const uint4& x) {
      *reinterpret_cast<uint2*>(row) = number ? codes_of<BF, E4M3>(x, r) : make_uint2(0, 0);
    };
    uint8_t* out0 = out + (r0 + rl) * c.token_stride;
    const int64_t out_step = per * c.token_stride;
#pragma unroll
    for (int s = 0; s < kHold; ++s) {
      const int row = r0 + s * per + rl;
      if (has(row)) put(out0 + s * out_step, w[s]);
    }
    for (int row = r0 + kHold * per + rl; row < r1; row += per)
      if (has(row)) put(out + row * c.token_stride, load(tok0 + row * step, row));
  }
}

// The values of all pages: a block takes a head's part of a page at a time, a thread eight
// columns of a slot (so that a warp's stores of 16 bits are whole lines: with sixteen, two
// stores of half a sector pair each, L1 was the limit), four of them on their way at once.
template <bool E4M3, int DT>
__global__ void __launch_bounds__(256) paged8_dequantize_kernel(const Cache c, void* k_out, void* v_out) {
  const int chunks = c.head_dim / 8, n = c.page_size * chunks;
  const bool is_v = blockIdx.y != 0;
  const uint8_t* src = is_v ? c.v : c.k;
  const float* scales = is_v ? c.v_scales : c.k_scales;
  char* out = reinterpret_cast<char*>(is_v ? v_out : k_out);
  constexpr int kAhead = 4, kBytes = DT == TS_F32 ? 32 : 16;       // of a thread's eight values
  const int off0 = threadIdx.x / chunks, ch0 = threadIdx.x - off0 * chunks;
  const int off_step = blockDim.x / chunks, ch_step = blockDim.x - off_step * chunks;
  for (int64_t ph = blockIdx.x; ph < (int64_t)c.num_pages * c.n_kv; ph += gridDim.x) {
    const int page = (int)(ph / c.n_kv), h = (int)(ph - (int64_t)page * c.n_kv);
    const uint8_t* rows = src + row_at(c, page, h, 0);
    const float* sc = scales + ph * c.blocks;
    int off = off0, ch = ch0;
    for (int i = threadIdx.x; i < n; i += kAhead * blockDim.x) {
      uint2 w[kAhead];
      float s[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (i + k * (int)blockDim.x < n) {
          w[k] = __ldg(reinterpret_cast<const uint2*>(rows + off * c.token_stride + ch * 8));
          s[k] = __ldg(sc + off / c.block);
        }
        off += off_step;
        ch += ch_step;
        if (ch >= chunks) {
          ch -= chunks;
          ++off;
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int at = i + k * (int)blockDim.x;
        if (at >= n) break;
        const Two ss = two(s[k], s[k]);
        float x[4], y[4];
        decode4<E4M3>(w[k].x, x);
        decode4<E4M3>(w[k].y, y);
        const float2 f[4] = {both(mul2(two(x[0], x[1]), ss)), both(mul2(two(x[2], x[3]), ss)), both(mul2(two(y[0], y[1]), ss)),
                             both(mul2(two(y[2], y[3]), ss))};
        uint4* p = reinterpret_cast<uint4*>(out + (ph * n + at) * kBytes);
        if constexpr (DT == TS_F32) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            p[e] = make_uint4(__float_as_uint(f[2 * e].x), __float_as_uint(f[2 * e].y), __float_as_uint(f[2 * e + 1].x),
                              __float_as_uint(f[2 * e + 1].y));
        } else {
          constexpr bool kBF = DT == TS_BF16;
          *p = make_uint4(pack2<kBF>(f[0].x, f[0].y), pack2<kBF>(f[1].x, f[1].y), pack2<kBF>(f[2].x, f[2].y),
                          pack2<kBF>(f[3].x, f[3].y));
        }
      }
    }
  }
}

int make_cache(const ts_paged_cache8* p, Cache* o) {
  TS_REQUIRE(p != nullptr, "NULL cache");
  TS_REQUIRE(p->batch == 0 || (p->k_pages && p->v_pages && p->k_scales && p->v_scales && p->page_table && p->seq_lens),
             "NULL pointer in the cache");
  TS_UNSUPPORTED(p->code == TS_CACHE_INT8 || p->code == TS_CACHE_E4M3, "the cache holds int8 or e4m3");
  TS_REQUIRE(p->batch >= 0 && p->n_kv > 0 && p->page_size > 0 && p->block > 0 && p->num_pages >= 0 &&
                 (p->batch == 0 || (p->num_pages > 0 && p->max_pages > 0)),
             "bad cache sizes");
  TS_UNSUPPORTED(p->head_dim % 16 == 0 && p->head_dim >= 16 && p->head_dim <= 256,
                 "head_dim must be a multiple of 16, <= 256");
  TS_UNSUPPORTED(p->block % 16 == 0 && p->page_size % p->block == 0,
                 "a page must hold whole blocks, and a block a multiple of 16 slots");
  TS_REQUIRE((int64_t)p->max_pages * p->page_size <= (int64_t)1 << 30, "more than 2^30 slots per sequence");
  TS_REQUIRE(is_aligned(p->k_pages, 16) && is_aligned(p->v_pages, 16) && p->page_stride % 16 == 0 &&
                 p->head_stride % 16 == 0 && p->token_stride % 16 == 0,
             "cache rows must be 16-byte aligned");
  o->k = reinterpret_cast<uint8_t*>(p->k_pages);
  o->v = reinterpret_cast<uint8_t*>(p->v_pages);
  o->page_stride = p->page_stride;
  o->head_stride = p->head_stride;
  o->token_stride = p->token_stride;
  o->k_scales = p->k_scales;
  o->v_scales = p->v_scales;
  o->table = p->page_table;
  o->table_stride = p->table_stride;
  o->seq_lens = p->seq_lens;
  o->batch = p->batch;
  o->n_kv = p->n_kv;
  o->head_dim = p->head_dim;
  o->page_size = p->page_size;
  o->num_pages = p->num_pages;
  o->max_pages = p->max_pages;
  o->block = p->block;
  o->blocks = p->page_size / p->block;
  return TS_OK;
}

template <bool BF, bool E4M3>
static void append(const AppendArgs& a, dim3 grid, cudaStream_t st) {
  if (a.cos_t != nullptr) paged8_append_kernel<BF, E4M3, true><<<grid, 256, 0, st>>>(a);
  else paged8_append_kernel<BF, E4M3, false><<<grid, 256, 0, st>>>(a);
}

int launch_append(const AppendArgs& a, int dtype, int code, int64_t most, cudaStream_t st) {
  const int64_t slots = std::min<int64_t>(most, (int64_t)a.c.max_pages * a.c.page_size);
  const int64_t items = ((slots + a.c.block - 1) / a.c.block + 1) * a.c.n_kv * 2;
  TS_UNSUPPORTED(a.c.batch <= 65535 && items < (int64_t)1 << 30, "too many sequences or tokens in one call");
  const dim3 grid((unsigned)std::max<int64_t>(1, std::min<int64_t>((items + 7) / 8, (16 * sm_count() + a.c.batch - 1) / a.c.batch)),
                  (unsigned)a.c.batch);
  if (dtype == TS_BF16) code == TS_CACHE_E4M3 ? append<true, true>(a, grid, st) : append<true, false>(a, grid, st);
  else code == TS_CACHE_E4M3 ? append<false, true>(a, grid, st) : append<false, false>(a, grid, st);
  TS_LAUNCH_CHECK();
  return TS_OK;
}

}  // namespace paged8
}  // namespace ts

using namespace ts;
using namespace ts::paged8;

extern "C" int ts_paged8_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                int kv_dtype, int64_t tokens, const int32_t* offsets, const int32_t* n_new,
                                const ts_paged_cache8* cache, const int64_t* first, const float* rope_cos,
                                const float* rope_sin, int64_t rope_rows, void* stream) {
  AppendArgs a;
  const int rc = make_cache(cache, &a.c);
  if (rc != TS_OK) return rc;
  TS_REQUIRE(tokens >= 0, "bad tokens");
  TS_UNSUPPORTED(kv_dtype == TS_F16 || kv_dtype == TS_BF16, "k and v must be fp16 or bf16");
  if (a.c.batch == 0 || tokens == 0) return TS_OK;     // (there may be no memory behind the pointers)
  TS_REQUIRE(k && v && k_strides && v_strides, "NULL pointer");
  TS_REQUIRE((rope_cos == nullptr) == (rope_sin == nullptr), "rope_cos and rope_sin come both or neither");
  for (int i = 0; i < 3; ++i)
    TS_REQUIRE(k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0, "k and v rows must be 16-byte aligned");
  TS_REQUIRE(is_aligned(k, 16) && is_aligned(v, 16), "k and v must be 16-byte aligned");
  a.k = reinterpret_cast<const uint16_t*>(k);
  a.v = reinterpret_cast<const uint16_t*>(v);
  a.kb = k_strides[0]; a.kt = k_strides[1]; a.kh = k_strides[2];
  a.vb = v_strides[0]; a.vt = v_strides[1]; a.vh = v_strides[2];
  a.tokens = tokens;
  a.offsets = offsets;
  a.n_new = n_new;
  a.first = first;
  a.cos_t = rope_cos;
  a.sin_t = rope_sin;
  a.rope_rows = rope_rows;
  return launch_append(a, kv_dtype, cache->code, tokens, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int ts_paged8_dequantize(const ts_paged_cache8* cache, void* k, void* v, int out_dtype, void* stream) {
  Cache c;
  const int rc = make_cache(cache, &c);
  if (rc != TS_OK) return rc;
  TS_UNSUPPORTED(out_dtype == TS_F16 || out_dtype == TS_BF16 || out_dtype == TS_F32, "unknown output type %d", out_dtype);
  if ((int64_t)c.num_pages * c.n_kv * c.page_size == 0) return TS_OK;
  TS_REQUIRE(c.k && c.v && c.k_scales && c.v_scales && k && v && is_aligned(k, 16) && is_aligned(v, 16),
             "NULL or unaligned pointer");
  const dim3 grid((unsigned)std::min<int64_t>((int64_t)c.num_pages * c.n_kv, (int64_t)1 << 24), 2);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto run = [&](auto kernel) { kernel<<<grid, 256, 0, st>>>(c, k, v); };
  if (cache->code == TS_CACHE_E4M3) {
    if (out_dtype == TS_BF16) run(paged8_dequantize_kernel<true, TS_BF16>);
    else if (out_dtype == TS_F16) run(paged8_dequantize_kernel<true, TS_F16>);
    else run(paged8_dequantize_kernel<true, TS_F32>);
  } else {
    if (out_dtype == TS_BF16) run(paged8_dequantize_kernel<false, TS_BF16>);
    else if (out_dtype == TS_F16) run(paged8_dequantize_kernel<false, TS_F16>);
    else run(paged8_dequantize_kernel<false, TS_F32>);
  }
  TS_LAUNCH_CHECK();
  return TS_OK;
}
