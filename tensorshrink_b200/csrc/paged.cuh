// Addressing of the paged key-value cache, shared by its kernels.
//
// A slot of a sequence is one cached token. Slot s lives in page
// table[s / page_size] at offset s % page_size; a page holds page_size tokens
// of every kv head. A table entry outside [0, num_pages) means that the slot
// has no memory: nothing is read from or written to it.
#pragma once

#include "sm100.cuh"

namespace ts {
namespace paged {

struct Cache {
  char* k;
  char* v;
  int64_t page_stride, head_stride, token_stride;   // elements, the same for k and v
  const int32_t* table;
  int64_t table_stride;
  int32_t* seq_lens;
  float* scores;       // [num_pages, n_kv, page_size] fp32, contiguous, or NULL
  int32_t* slot_pos;   // the same of int32, or NULL
  int batch, n_kv, head_dim, page_size, num_pages, max_pages;
};

// Checks the description of a cache and fills the device view.
int make_cache(const ts_paged_cache* c, Cache* out);
int log2_of(int v);   // -1 of anything but a power of two

__device__ __forceinline__ int64_t capacity(const Cache& c) { return (int64_t)c.max_pages * c.page_size; }

// Page of slot s of sequence b, or -1 when the slot has no memory.
__device__ __forceinline__ int page_of(const Cache& c, int b, int s) {
  const int i = s / c.page_size;
  if (i >= c.max_pages) return -1;
  const int p = c.table[b * c.table_stride + i];
  return (unsigned)p < (unsigned)c.num_pages ? p : -1;
}

// Element offset of (page, head, offset in the page) in k and v.
__device__ __forceinline__ int64_t row_at(const Cache& c, int page, int h, int off) {
  return (int64_t)page * c.page_stride + (int64_t)h * c.head_stride + (int64_t)off * c.token_stride;
}

// Index of (page, head, offset) in scores and slot_pos.
__device__ __forceinline__ int64_t stat_at(const Cache& c, int page, int h, int off) {
  return ((int64_t)page * c.n_kv + h) * c.page_size + off;
}

template <bool BF>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Rotary embedding of the pair (x1, x2) = (x[i], x[i + D / 2]): products and
// sums rounded to fp32 one by one, as separate tensor operations round them,
// so that cached keys equal those of an unfused model bit for bit.
__device__ __forceinline__ float2 rotate(float x1, float x2, float c, float s) {
  return make_float2(__fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s)), __fadd_rn(__fmul_rn(x1, s), __fmul_rn(x2, c)));
}

// Workspace of the serving kernels on a stream: first kCounters ints, zero
// between calls, whose places no call uses for anything else; scratch behind.
constexpr size_t kCounters = 65536;
constexpr size_t kCounterBytes = kCounters * 4;

}  // namespace paged
}  // namespace ts
