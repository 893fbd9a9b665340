// Page tables and slot maps from request lengths, and the pages of sequences that
// are cut back.
//
// One launch of one cluster: each CTA takes a run of the sequences, a warp one of them at
// a time (its lanes look at neighbouring entries of the table). The pages that the
// sequences need become places in the pool by a sum over the CTA's run and,
// through distributed shared memory, over those of the CTAs in front; then the
// warps write the entries, and after a barrier of the cluster all threads write the slots of
// the packed tokens, finding each token's sequence by bisection in shared memory. Bound by
// latency: a chain of a few loads and barriers. A small batch takes one CTA. 8 sequences that take
// one token each: 6 us, and 4 us for the release; 256, eight of them prompts of up to 8000 tokens:
// 13.5 and 5 us.
#include <algorithm>

#include "gemm.cuh"
#include "paged.cuh"

namespace ts {
namespace paged {

constexpr int kTableThreads = 1024;
constexpr int kTableWarps = kTableThreads / 32;
constexpr int kTableCtas = 8;              // of the cluster
constexpr int kMaxSequences = 8192;      // (three words of each in shared memory)

struct TableArgs {
  int32_t* free_pages;
  int32_t* n_free;
  int capacity;
  int32_t* table;
  int64_t table_stride;
  int32_t* seq_lens;
  int batch, max_pages, page_size, num_pages;
  int page_shift;
  int per;                 // sequences of a CTA
  const int32_t* n_new;    // or keep
  const int64_t* first;
  int64_t tokens;
  int32_t* granted;
  int32_t* offsets;
  int64_t* slots;
  int64_t* positions;
  int32_t* sequences;
};

__device__ __forceinline__ int64_t ld_cluster64(uint32_t addr) {
  int64_t v;
  asm volatile("ld.shared::cluster.s64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ int cluster_ctas() {
  uint32_t n;
  asm volatile("mov.u32 %0, %cluster_nctaid.x;" : "=r"(n));
  return (int)n;
}

__device__ __forceinline__ bool is_page(const TableArgs& a, int p) { return (unsigned)p < (unsigned)a.num_pages; }
__device__ __forceinline__ int64_t pages_for(const TableArgs& a, int64_t slots) {
  return a.page_shift >= 0 ? (slots + a.page_size - 1) >> a.page_shift : (slots + a.page_size - 1) / a.page_size;
}

// Entries [p0, p1) of a row of the table whose being a page is `want`, counted by a warp.
__device__ __forceinline__ int count_entries(const TableArgs& a, const int32_t* row, int p0, int p1, bool want) {
  const int lane = threadIdx.x & 31;
  int n = 0;
  for (int p = p0 + lane; p < p1; p += 128) {
    int e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = p + 32 * i < p1 ? row[p + 32 * i] : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) n += p + 32 * i < p1 && is_page(a, e[i]) == want;
  }
  return __reduce_add_sync(0xffffffffu, n);
}

// In place: the sums in front of each of v[0 .. n), and the sum of all in total. By one warp.
__device__ __forceinline__ void exclusive_sums(int64_t* v, int n, int64_t* total) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int64_t x = i0 + lane < n ? v[i0 + lane] : 0;
    int64_t s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    if (i0 + lane < n) v[i0 + lane] = before + s - x;
    before += __shfl_sync(0xffffffffu, s, 31);
  }
  if (lane == 0) *total = before;
}

// What the CTAs in front of this one have in `total`, and what all have, in out[0], out[1]. By one warp, a
// lane a CTA.
__device__ __forceinline__ void cluster_sums(const int64_t* total, int64_t* out) {
  const int lane = threadIdx.x & 31, rank = (int)cta_rank();
  const int64_t x = lane < cluster_ctas() ? ld_cluster64(map_cta(smem_u32(total), lane)) : 0;
  int64_t front = lane < rank ? x : 0, all = x;
  static_assert(kTableCtas <= 8, "lanes");
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    front += __shfl_xor_sync(0xffffffffu, front, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  if (lane == 0) {
    out[0] = front;
    out[1] = all;
  }
}

__global__ void __launch_bounds__(kTableThreads, 1) paged_reserve_kernel(const TableArgs a) {
  extern __shared__ int64_t sums[];                 // [per] pages of the run's sequences, [per] tokens; [batch + 1] offsets
  __shared__ int64_t total[2], popped, across[2][2];
  int64_t* tokens = sums + a.per;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cta_rank();
  const int b0 = rank * a.per, mine = max(0, min(a.per, a.batch - b0));
  const int n_free = max(0, min(*a.n_free, a.capacity));
  const int64_t slots_max = (int64_t)a.max_pages * a.page_size;
  auto takes = [&](int len, int n) { return n > 0 && len >= 0 && len + (int64_t)n <= slots_max; };
  if (threadIdx.x == 0) popped = 0;
  for (int i = warp; i < mine; i += kTableWarps) {
    const int b = b0 + i, len = a.seq_lens[b], n = max(0, a.n_new[b]);
    int need = 0;
    if (takes(len, n)) {
      const int p0 = len / a.page_size, p1 = (int)pages_for(a, len + (int64_t)n);
      need = count_entries(a, a.table + b * a.table_stride, p0, p1, false);
    }
    if (lane == 0) {
      sums[i] = need;
      tokens[i] = n;
    }
  }
  __syncthreads();
  if (warp < 2) exclusive_sums(warp == 0 ? sums : tokens, mine, total + warp);
  cluster_sync();
  if (warp < 2) cluster_sums(total + warp, across[warp]);
  __syncthreads();
  const int64_t front = across[0][0], front_tokens = across[1][0];
  // the entries
  for (int i = warp; i < mine; i += kTableWarps) {
    const int b = b0 + i, len = a.seq_lens[b], n = max(0, a.n_new[b]);
    const int64_t at = front + sums[i], end = front + (i + 1 < mine ? sums[i + 1] : total[0]);
    const bool served = takes(len, n) && (at == end || end <= n_free);
    if (served && at < end) {
      int32_t* row = a.table + b * a.table_stride;
      const int p0 = len / a.page_size, p1 = (int)pages_for(a, len + (int64_t)n);
      int k = (int)at;                                 // (end is at most n_free)
      for (int q = p0 + lane; q - lane < p1; q += 128) {
        int to[4];                                     // place in the pool of each empty entry
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i] = q + 32 * i < p1 ? row[q + 32 * i] : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool empty = q + 32 * i < p1 && !is_page(a, to[i]);
          const unsigned mask = __ballot_sync(0xffffffffu, empty);
          to[i] = empty ? n_free - 1 - (k + __popc(mask & ((1u << lane) - 1))) : -1;
          k += __popc(mask);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (to[i] >= 0) row[q + 32 * i] = a.free_pages[to[i]];
      }
    }
    if (lane == 0) {
      a.granted[b] = served ? n : 0;
      const int64_t t0 = front_tokens + tokens[i], t1 = front_tokens + (i + 1 < mine ? tokens[i + 1] : total[1]);
      a.offsets[b] = (int32_t)min(t0, (int64_t)INT32_MAX);
      if (b == a.batch - 1) a.offsets[a.batch] = (int32_t)min(t1, (int64_t)INT32_MAX);
      if (served && at < end) atomicMax(reinterpret_cast<unsigned long long*>(&popped), (unsigned long long)end);
    }
  }
  cluster_sync();                                    // the entries, counts and offsets are everybody's
  int* off = reinterpret_cast<int*>(sums + 2 * a.per);   // [batch + 1]
  int* len_of = off + a.batch + 1;                       // [batch] cached tokens, -1 of a sequence that got nothing
  for (int i = threadIdx.x; i <= a.batch; i += kTableThreads) {
    off[i] = __ldcg(a.offsets + i);
    if (i < a.batch) len_of[i] = __ldcg(a.granted + i) > 0 ? a.seq_lens[i] : -1;
  }
  if (rank == 0 && warp == 0) {
    // (served sequences need the pool's first pages: as many as the last of them ends at)
    int64_t top = 0;
    for (int i = 0; i < cluster_ctas(); ++i) top = max(top, ld_cluster64(map_cta(smem_u32(&popped), i)));
    if (lane == 0) *a.n_free = n_free - (int)top;
  }
  __syncthreads();
  // kAhead tokens of a thread at a time, so that their look-ups in the table overlap
  constexpr int kAhead = 4;
  const int64_t step = (int64_t)cluster_ctas() * kTableThreads;
  for (int64_t t0 = (int64_t)rank * kTableThreads + threadIdx.x; t0 < a.tokens; t0 += kAhead * step) {
    int b[kAhead], s[kAhead], page[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t t = t0 + k * step;
      b[k] = s[k] = page[k] = -1;
      if (t >= a.tokens || t >= off[a.batch]) continue;
      // the last sequence that starts at t or in front of it (those without tokens start where the next one does)
      int lo = 0;
      for (int hi = a.batch - 1; lo < hi;) {
        const int mid = (lo + hi + 1) >> 1;
        if (off[mid] <= t) lo = mid; else hi = mid - 1;
      }
      b[k] = lo;
      if (len_of[lo] < 0) continue;
      s[k] = len_of[lo] + (int)(t - off[lo]);
      page[k] = __ldcg(a.table + lo * a.table_stride + (a.page_shift >= 0 ? s[k] >> a.page_shift : s[k] / a.page_size));
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t t = t0 + k * step;
      if (t >= a.tokens) break;
      const bool has = is_page(a, page[k]);
      const int in_page = a.page_shift >= 0 ? s[k] & (a.page_size - 1) : s[k] % a.page_size;
      a.slots[t] = has ? (int64_t)page[k] * a.page_size + in_page : -1;
      a.positions[t] = !has ? 0 : a.first != nullptr ? a.first[b[k]] + (t - off[b[k]]) : s[k];
      a.sequences[t] = b[k];
    }
  }
  cluster_sync();                                    // nobody leaves while its sums may be read
}

__global__ void __launch_bounds__(kTableThreads, 1) paged_release_kernel(const TableArgs a) {
  extern __shared__ int64_t sums[];                 // [per] pages of the run's sequences
  __shared__ int64_t total, across[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b0 = (int)cta_rank() * a.per, mine = max(0, min(a.per, a.batch - b0));
  const int n_free = max(0, min(*a.n_free, a.capacity));
  auto first_page = [&](int len, int keep) { return (int)min((int64_t)a.max_pages, pages_for(a, max(0, min(len, keep)))); };
  for (int i = warp; i < mine; i += kTableWarps) {
    const int b = b0 + i, keep = a.n_new[b];
    int n = 0;
    if (keep >= 0) n = count_entries(a, a.table + b * a.table_stride, first_page(a.seq_lens[b], keep), a.max_pages, true);
    if (lane == 0) sums[i] = n;
  }
  __syncthreads();
  if (warp == 0) exclusive_sums(sums, mine, &total);
  cluster_sync();
  if (warp == 0) cluster_sums(&total, across);
  __syncthreads();
  const int64_t front = across[0], all = across[1];
  for (int i = warp; i < mine; i += kTableWarps) {
    const int b = b0 + i, keep = a.n_new[b];
    if (keep < 0) continue;
    int32_t* row = a.table + b * a.table_stride;
    const int len = a.seq_lens[b];
    int64_t at = n_free + front + sums[i];
    const int64_t end = n_free + front + (i + 1 < mine ? sums[i + 1] : total);
    for (int q = first_page(len, keep) + lane; at < end && q - lane < a.max_pages; q += 128) {
      int e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = q + 32 * i < a.max_pages ? row[q + 32 * i] : -1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool full = is_page(a, e[i]);
        const unsigned mask = __ballot_sync(0xffffffffu, full);
        if (full) {
          const int64_t to = at + __popc(mask & ((1u << lane) - 1));
          if (to < a.capacity) a.free_pages[to] = e[i];   // (more pages than the pool has: some were shared)
          row[q + 32 * i] = -1;
        }
        at += __popc(mask);
      }
    }
    __syncwarp();
    if (lane == 0 && len > keep) a.seq_lens[b] = keep;
  }
  if (cta_rank() == 0 && threadIdx.x == 0) *a.n_free = (int)min((int64_t)a.capacity, n_free + all);
  cluster_sync();                                    // nobody leaves while its sums may be read
}

static int make_table(const ts_page_pool* pool, const ts_page_table* t, const int32_t* per_sequence, TableArgs* a) {
  TS_REQUIRE(pool != nullptr && t != nullptr, "NULL pool or table");
  TS_REQUIRE(pool->capacity >= 0 && t->batch >= 0 && t->page_size > 0 && t->max_pages >= 0 && t->num_pages >= 0, "bad sizes");
  TS_UNSUPPORTED(t->batch <= kMaxSequences, "more than %d sequences", kMaxSequences);
  TS_REQUIRE((int64_t)t->max_pages * t->page_size <= (int64_t)1 << 30, "more than 2^30 slots per sequence");
  TS_REQUIRE(t->batch == 0 || (pool->n_free && (pool->capacity == 0 || pool->free_pages) && t->seq_lens && per_sequence &&
                               (t->max_pages == 0 || t->table)),
             "NULL pointer");
  *a = TableArgs{};
  a->free_pages = pool->free_pages;
  a->n_free = pool->n_free;
  a->capacity = pool->capacity;
  a->table = t->table;
  a->table_stride = t->table_stride;
  a->seq_lens = t->seq_lens;
  a->batch = t->batch;
  a->max_pages = t->max_pages;
  a->page_size = t->page_size;
  a->num_pages = t->num_pages;
  a->page_shift = log2_of(t->page_size);
  a->n_new = per_sequence;
  return TS_OK;
}

template <typename K>
static int launch_tables(K k, TableArgs& a, int64_t work, size_t more, cudaStream_t st) {
  // one CTA where each of its warps has a sequence and its threads a few tokens
  const int ctas = a.batch <= kTableWarps && work <= 2 * kTableThreads ? 1 : kTableCtas;
  a.per = (a.batch + ctas - 1) / ctas;
  const size_t smem = (size_t)a.per * 16 + more;
  if (smem > 48 * 1024) {
    const int rc = open_smem(reinterpret_cast<const void*>(k));
    if (rc != TS_OK) return rc;
  }
  TS_CUDA_TRY(launch_after(k, ctas, kTableThreads, smem, st, 0, ctas, a));
  TS_LAUNCH_CHECK();
  return TS_OK;
}

}  // namespace paged
}  // namespace ts

using namespace ts;
using namespace ts::paged;

extern "C" int ts_paged_reserve(const ts_page_pool* pool, const ts_page_table* table, const int32_t* n_new,
                                const int64_t* first, int64_t tokens, int32_t* granted, int32_t* offsets, int64_t* slots,
                                int64_t* positions, int32_t* sequences, void* stream) {
  TableArgs a;
  const int rc = make_table(pool, table, n_new, &a);
  if (rc != TS_OK) return rc;
  TS_REQUIRE(tokens >= 0 && tokens < (int64_t)1 << 31, "bad tokens");
  TS_REQUIRE(a.batch > 0, "no sequences");
  TS_REQUIRE(granted && offsets && (tokens == 0 || (slots && positions && sequences)), "NULL pointer");
  a.first = first;
  a.tokens = tokens;
  a.granted = granted;
  a.offsets = offsets;
  a.slots = slots;
  a.positions = positions;
  a.sequences = sequences;
  return launch_tables(paged_reserve_kernel, a, tokens, (size_t)(2 * a.batch + 1) * 4, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int ts_paged_release(const ts_page_pool* pool, const ts_page_table* table, const int32_t* keep, void* stream) {
  TableArgs a;
  const int rc = make_table(pool, table, keep, &a);
  if (rc != TS_OK) return rc;
  if (a.batch == 0 || a.max_pages == 0) return TS_OK;
  return launch_tables(paged_release_kernel, a, (int64_t)a.batch * a.max_pages / 4, 0, reinterpret_cast<cudaStream_t>(stream));
}
