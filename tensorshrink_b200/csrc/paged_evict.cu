// Eviction from a paged key-value cache by accumulated attention weight.
//
// For each sequence longer than `budget` and each kv head, `budget` slots
// stay: those whose position is among the `recent` newest, then those of the
// largest score (ties to the lowest slot; a NaN score counts as -inf, and
// a slot without memory goes first). Kept slots at or behind `budget` move
// into the holes before it, both taken in ascending order, with k, v, score
// and position; the sequence's length becomes `budget`. Attention does not
// depend on the order of slots, so nothing else has to move: after one new
// token a single slot does, where a shift that keeps the order would rewrite
// most of the cache. Sources lie behind `budget` and targets before it, so
// all moves of a call are independent of one another.
//
// select: one CTA per (sequence, kv head) finds the budget-th largest key by
// radix selection over monotone 32-bit keys (three digits of 11, 11 and 10
// bits, histograms in shared memory) and lists holes and movers by block
// scans. move: a warp copies eight slots at a time, 16 bytes per lane and row.
// Where a head can have only few movers (a token in, a token out), the select
// CTA moves them itself and there is no second kernel.
// What bounds them: select reads 8 bytes per slot and is latency-bound at one
// CTA per head (1025 slots 9.6 us with its one move, 8192 slots 15 us); move is
// DRAM traffic of the moved slots only (16 sequences cut from 8192 to 4096 slots
// of 8 heads of 128 columns: 25 us, lists and pages looked up on the way).
#include <algorithm>
#include <climits>

#include "paged.cuh"

namespace ts {
namespace paged {

constexpr int kSelThreads = 1024;
constexpr int kBins = 2048;
constexpr int kMoveWarps = 8;
constexpr int kInline = 64;            // moves that a select CTA does itself
constexpr int kMoves = 8;              // slots that a warp moves at a time
constexpr int kSmemKeys = 24 * 1024;   // slots of a select CTA in shared memory

struct EvictArgs {
  Cache c;
  int budget, recent;
  int* n_move;            // [batch * n_kv]
  int32_t* holes;         // [batch * n_kv][list]
  int32_t* movers;
  int list;
  uint32_t* keys;         // [batch * n_kv][2][cap]: keys and positions that do not fit shared memory
  int64_t cap;
  int smem_keys;          // slots whose keys and positions fit shared memory
  int page_shift;         // log2(page_size), or -1
  int* counters;          // [batch] heads of a sequence that are done (moves in the select CTA)
  int inline_moves;       // at most kInline moves a head: the select CTA does them itself
};

// Monotone key: larger scores have larger keys, -0 equals +0, NaN counts as -inf.
__device__ __forceinline__ uint32_t key_of(float s) {
  const uint32_t u = isnan(s) ? 0xFF800000u : __float_as_uint(s == 0.f ? 0.f : s);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive block scan of one int per thread; *sum receives the total.
__device__ __forceinline__ int block_scan(int v, int* sum, int* warp_tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  __syncthreads();
  if (lane == 31) warp_tot[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int w = lane < kSelThreads / 32 ? warp_tot[lane] : 0;
    int wi = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, wi, o);
      if (lane >= o) wi += t;
    }
    warp_tot[lane] = wi - w;
    if (lane == 31) warp_tot[32] = wi;
  }
  __syncthreads();
  *sum = warp_tot[32];
  return warp_tot[warp] + inc - v;
}

// Moves first .. n - 1 of a head's list, kMoves of them per step, by one warp;
// `to` is the warp's place for 2 kMoves offsets.
__device__ __forceinline__ void move_slots(const Cache& c, int b, int h, const int32_t* lh, const int32_t* lm, int first,
                                           int n, int step, int64_t* to) {
  const int lane = threadIdx.x & 31, chunks = c.head_dim / 8;
  for (int i0 = first; i0 < n; i0 += step) {
    // lane k looks up target k, lane k + 16 source k
    int64_t row_off = -1, stat = 0;
    if ((lane & 15) < kMoves && i0 + (lane & 15) < n) {
      const int slot = (lane < 16 ? lh : lm)[i0 + (lane & 15)];
      const int page = page_of(c, b, slot), off = slot % c.page_size;
      if (page >= 0) {
        row_off = row_at(c, page, h, off) * 2;
        stat = stat_at(c, page, h, off);
      }
    }
    const int64_t src_stat = __shfl_down_sync(0xffffffffu, stat, 16);
    const int64_t src_off = __shfl_down_sync(0xffffffffu, row_off, 16);
    if (lane < kMoves && row_off >= 0 && src_off >= 0) {
      c.scores[stat] = c.scores[src_stat];
      c.slot_pos[stat] = c.slot_pos[src_stat];
    }
    const unsigned moves = __ballot_sync(0xffffffffu, lane < kMoves && row_off >= 0 && src_off >= 0);
    // the rows' places, read back by every lane
    int64_t* from = to + kMoves;
    if ((lane & 15) < kMoves) to[(lane >> 4) * kMoves + (lane & 15)] = row_off;
    __syncwarp();
    for (int ch = lane; ch < 2 * chunks; ch += 32) {
      char* base = (ch < chunks ? c.k : c.v) + (ch < chunks ? ch : ch - chunks) * 16;
      uint4 w[kMoves];
#pragma unroll
      for (int k = 0; k < kMoves; ++k)
        if ((moves >> k) & 1) w[k] = *reinterpret_cast<const uint4*>(base + from[k]);
#pragma unroll
      for (int k = 0; k < kMoves; ++k)
        if ((moves >> k) & 1) *reinterpret_cast<uint4*>(base + to[k]) = w[k];
    }
    __syncwarp();
  }
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
  extern __shared__ uint32_t skeys[];
  __shared__ __align__(16) int hist[kBins];
  static_assert(kSelThreads / 32 * 2 * kMoves * 8 <= sizeof(int) * kBins, "the moves' offsets lie over the histogram");
  __shared__ int warp_tot[33];
  __shared__ int s_newest, s_digit, s_left;
  pdl_launch_dependents();
  const Cache& c = a.c;
  const int row = blockIdx.x, b = row / c.n_kv, h = row - b * c.n_kv, tid = threadIdx.x;
  const int n = (int)min((int64_t)max(c.seq_lens[b], 0), capacity(c));
  if (n <= a.budget) {   // (so are the sequence's other heads)
    if (tid == 0) a.n_move[row] = 0;
    return;
  }
  uint32_t* keys = n <= a.smem_keys ? skeys : a.keys + (int64_t)row * a.cap * 2;
  int32_t* pos = reinterpret_cast<int32_t*>(keys + (n <= a.smem_keys ? a.smem_keys : a.cap));

  // keys and positions, four slots of a thread in flight; the newest position
  if (tid == 0) s_newest = INT_MIN;
  __syncthreads();
  int newest = INT_MIN;
  for (int i0 = tid; i0 < n; i0 += 4 * kSelThreads) {
    int64_t at[4];
    float sc[4];
    int po[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * kSelThreads, pg = a.page_shift >= 0 ? i >> a.page_shift : i / c.page_size;
      const int page = i < n ? c.table[b * c.table_stride + pg] : -1;
      at[k] = (unsigned)page < (unsigned)c.num_pages ? stat_at(c, page, h, i - pg * c.page_size) : -1;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at[k] >= 0) {
        sc[k] = c.scores[at[k]];
        po[k] = c.slot_pos[at[k]];
      }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * kSelThreads;
      if (i >= n) break;
      // a slot without memory: key 0, below every score's, and never recent
      keys[i] = at[k] >= 0 ? key_of(sc[k]) : 0;
      pos[i] = at[k] >= 0 ? po[k] : INT_MIN;
      if (at[k] >= 0) newest = max(newest, po[k]);
    }
  }
  newest = __reduce_max_sync(0xffffffffu, newest);
  if ((tid & 31) == 0) atomicMax(&s_newest, newest);
  __syncthreads();
  const int64_t limit = (int64_t)s_newest - a.recent;
  for (int i = tid; i < n; i += kSelThreads)
    if ((int64_t)pos[i] > limit && keys[i] != 0) keys[i] = 0xFFFFFFFFu;   // recent: above any score

  // radix selection of the budget-th largest key
  uint32_t prefix = 0, mask = 0;
  int left = a.budget;   // how many of the keys with this prefix stay
  const int shifts[3] = {21, 10, 0};
  const int widths[3] = {11, 11, 10};
#pragma unroll
  for (int d = 0; d < 3; ++d) {
    const int bins = 1 << widths[d];
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSelThreads) {
      const uint32_t k = keys[i];
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shifts[d]) & (bins - 1)], 1);
    }
    __syncthreads();
    // thread t holds the two bins 2047 - 2t and 2046 - 2t: a scan from the top
    const int hi = kBins - 1 - 2 * tid;
    const int n1 = hist[hi], n0 = hist[hi - 1];
    int total;
    const int before = block_scan(n1 + n0, &total, warp_tot);
    if (before < left && left <= before + n1) {
      s_digit = hi;
      s_left = left - before;
    } else if (before + n1 < left && left <= before + n1 + n0) {
      s_digit = hi - 1;
      s_left = left - before - n1;
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shifts[d];
    mask |= (uint32_t)(bins - 1) << shifts[d];
    left = s_left;
    __syncthreads();
  }

  // of the keys equal to the threshold the first `left` stay. Every thread
  // takes a run of slots (an odd number, so that their keys fall in
  // different banks).
  const int per = ((n + kSelThreads - 1) / kSelThreads) | 1;
  const int i0 = min(tid * per, n), i1 = min(i0 + per, n);
  int eq = 0;
  for (int i = i0; i < i1; ++i) eq += keys[i] == prefix;
  int dummy;
  const int eq0 = block_scan(eq, &dummy, warp_tot);
  int holes = 0, movers = 0, e = eq0;
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = keys[i];
    const bool keep = k > prefix || (k == prefix && e++ < left);
    if (i < a.budget) holes += !keep;
    else movers += keep;
  }
  int n_holes, n_movers;
  int at_h = block_scan(holes, &n_holes, warp_tot);
  int at_m = block_scan(movers, &n_movers, warp_tot);
  e = eq0;
  int32_t* lh = a.holes + (int64_t)row * a.list;
  int32_t* lm = a.movers + (int64_t)row * a.list;
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = keys[i];
    const bool keep = k > prefix || (k == prefix && e++ < left);
    if (i < a.budget) {
      if (!keep) lh[at_h++] = i;
    } else if (keep) {
      lm[at_m++] = i;
    }
  }
  if (!a.inline_moves) {
    if (tid == 0) a.n_move[row] = n_movers;   // == n_holes
    return;
  }
  __syncthreads();                            // the lists are written, the keys have been read
  move_slots(c, b, h, lh, lm, (tid >> 5) * kMoves, n_movers, kSelThreads / 32 * kMoves,
             reinterpret_cast<int64_t*>(hist) + (tid >> 5) * 2 * kMoves);
  // the last head of the sequence sets its length, which every head has read
  if (tid == 0 && atomicAdd(a.counters + b, 1) == c.n_kv - 1) {
    a.counters[b] = 0;
    c.seq_lens[b] = a.budget;
  }
}

__global__ void __launch_bounds__(kMoveWarps * 32) evict_move_kernel(const EvictArgs a) {
  __shared__ int64_t where[kMoveWarps][2 * kMoves];
  pdl_wait_primary();
  const Cache& c = a.c;
  const int row = blockIdx.y, b = row / c.n_kv, h = row - b * c.n_kv;
  const int n = a.n_move[row];
  const int32_t* lh = a.holes + (int64_t)row * a.list;
  const int32_t* lm = a.movers + (int64_t)row * a.list;
  move_slots(c, b, h, lh, lm, (blockIdx.x * kMoveWarps + (threadIdx.x >> 5)) * kMoves, n, gridDim.x * kMoveWarps * kMoves,
             where[threadIdx.x >> 5]);
  // nothing in this kernel reads the lengths, so they can be set here
  if (h == 0 && blockIdx.x == 0 && threadIdx.x == 0 && c.seq_lens[b] > a.budget) c.seq_lens[b] = a.budget;
}

struct EvictLayout {
  size_t n_move, holes, movers, keys, bytes;
  int64_t list;
  int smem_keys;
};

static EvictLayout evict_layout(const ts_paged_cache& p, int budget) {
  EvictLayout L;
  const int64_t cap = (int64_t)p.max_pages * p.page_size, rows = (int64_t)p.batch * p.n_kv;
  L.list = std::max<int64_t>(1, std::min<int64_t>(budget, cap - budget));
  L.smem_keys = (int)std::min<int64_t>(cap, kSmemKeys);
  L.n_move = kCounterBytes;
  L.holes = align_up(L.n_move + rows * 4, 256);
  L.movers = align_up(L.holes + rows * L.list * 4, 256);
  L.keys = align_up(L.movers + rows * L.list * 4, 256);
  L.bytes = L.keys + (cap > L.smem_keys ? (size_t)rows * cap * 8 : 0);
  return L;
}

}  // namespace paged
}  // namespace ts

using namespace ts;
using namespace ts::paged;

extern "C" size_t ts_paged_evict_workspace_size(const ts_paged_cache* cache, int budget) {
  if (cache == nullptr) return 0;
  return evict_layout(*cache, budget).bytes;
}

extern "C" int ts_paged_evict(const ts_paged_cache* cache, int budget, int recent, void* workspace,
                              size_t workspace_bytes, void* stream) {
  EvictArgs a;
  const int rc = make_cache(cache, &a.c);
  if (rc != TS_OK) return rc;
  TS_REQUIRE(a.c.batch == 0 || (a.c.scores != nullptr && a.c.slot_pos != nullptr), "eviction needs the cache's scores and slot_pos");
  TS_REQUIRE(budget > 0, "budget must be positive");
  TS_REQUIRE(recent >= 0 && recent <= budget, "recent must be in [0, budget]");
  const int64_t cap = (int64_t)a.c.max_pages * a.c.page_size;
  if (a.c.batch == 0 || cap <= budget) return TS_OK;
  const EvictLayout L = evict_layout(*cache, budget);
  if (workspace == nullptr || workspace_bytes < L.bytes) {
    set_error("workspace of %zu bytes, %zu needed", workspace_bytes, L.bytes);
    return TS_ERR_WORKSPACE;
  }
  TS_REQUIRE(is_aligned(workspace, 16), "workspace must be 16-byte aligned");
  char* ws = reinterpret_cast<char*>(workspace);
  a.budget = budget;
  a.recent = recent;
  a.n_move = reinterpret_cast<int*>(ws + L.n_move);
  a.holes = reinterpret_cast<int32_t*>(ws + L.holes);
  a.movers = reinterpret_cast<int32_t*>(ws + L.movers);
  a.list = (int)L.list;
  a.keys = reinterpret_cast<uint32_t*>(ws + L.keys);
  a.cap = cap;
  a.smem_keys = L.smem_keys;
  a.page_shift = log2_of(a.c.page_size);
  a.counters = reinterpret_cast<int*>(ws);
  a.inline_moves = L.list <= kInline && a.c.batch <= (int)kCounters ? 1 : 0;
  const int rows = a.c.batch * a.c.n_kv;
  TS_UNSUPPORTED(rows <= 65535, "too many heads in one call");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const size_t smem = (size_t)L.smem_keys * 8;
  static thread_local int configured_dev = -1;
  int dev = 0;
  TS_CUDA_TRY(cudaGetDevice(&dev));
  if (configured_dev != dev) {
    TS_CUDA_TRY(cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemKeys * 8));
    configured_dev = dev;
  }
  evict_select_kernel<<<rows, kSelThreads, smem, st>>>(a);
  TS_LAUNCH_CHECK();
  if (a.inline_moves) return TS_OK;
  const int per_row = (int)std::max<int64_t>(
      1, std::min<int64_t>((L.list + kMoveWarps * kMoves - 1) / (kMoveWarps * kMoves), (16 * sm_count() + rows - 1) / rows));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)per_row, (unsigned)rows);
  cfg.blockDim = dim3(kMoveWarps * 32);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];                         // (it waits for the selection by itself)
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  TS_CUDA_TRY(cudaLaunchKernelEx(&cfg, evict_move_kernel, a));
  TS_LAUNCH_CHECK();
  return TS_OK;
}
