// Attention of one token per sequence over a paged key-value cache of 8 bits.
//
//   s_t = scale q . (a_t k_t),   p = softmax(s),   o = sum_t p_t (b_t v_t)
//
// over the cached slots t, a_t and b_t the scales of t's block. The scales stay
// outside the products. Scores of integers are sums of products of bytes, q being three
// bytes of 24 bits (a head's power of two taken out), exact up to the last addition; those of
// e4m3 (and of wide groups, for registers) take the codes as fp16, exactly, and q as
// fp16 without its power of two. A score is the product of the sum with a_t. A weight
// enters the second product as p_t b_t over a power of two that is at least every
// |b_t| so far (the output is scaled along when it grows, as for the running
// maximum), as two terms of fp16, 22 bits (one term turned the last bits of bf16
// results).
//
// What bounds it: 2 len D bytes per kv head are read once, DRAM bandwidth does, but at
// half the bytes of a 16-bit cache the instructions per slot come close. So the
// slots are the MMA's 16 rows and the query heads its 8 columns (S^T = K Q^T,
// O^T = V^T P^T; groups of more than eight take two column tiles): for groups up
// to eight half the products, exponentials and registers of the other
// orientation. Codes come from shared memory as bytes, four of a register making two
// operand registers, with the order of columns inside a 16-column step permuted
// alike in q (scores) or in the output (whose accumulator rows g and g + 8 are the
// neighbouring columns 2 g and 2 g + 1); P turns from sums to operand by movmatrix. The running
// maximum follows only when a score passes it by 2^4, found by one vote, so that
// a tile usually needs no shuffles.
//
// The work is cut as in the 16-bit kernel (paged_split.cuh), in units of 128 slots, 32
// of each to a warp, which streams them through its own ring of stages: a TMA
// box each of k and v (two of 16 slots where pages are no multiple of 32), issued by
// one lane and complete on the stage's barrier, no CTA barrier in the loop. (Copies of 16 slots
// alone reach 5.1 TB/s where those of 32 reach 5.5.) Lane i of a warp looks up page and
// scales of its tile 32 j + i, three batches deep. Every wait is bounded; a warp whose
// wait runs out records it and stops.
//
// Measured (128 columns, 8 kv heads, other inputs each time, in a graph): 64 sequences of up to 8191 slots,
// 8 query heads to a kv head, int8, token-major pages, 102 us, 5.3 TB/s (a call 111, with one term for
// a weight 106); 4 of 32768, e4m3, fp16 results, 53 us, 5.1 TB/s; one of 512, 10.5 us, a chain of
// latencies and of first instruction fetches. Groups of more than eight heads, whose second column tile
// doubles the instructions of a slot, are bound by those: 16 heads, 32 sequences of up to 8000 slots
// 77 us (e4m3 71), 3.4 TB/s; 32 heads over one, each 16 of them reading the slots again, 32 of up to 20000 51 us for 81 MB.
#include <algorithm>

#include "gemm.cuh"
#include "paged8.cuh"
#include "paged_split.cuh"

namespace ts {
namespace paged8 {

using paged::choose_deal;
using paged::Deal;
using paged::ex2;
using paged::kCounterBytes;
using paged::kCounters;
using paged::kMaxPieces;
using paged::kRowCost;
using paged::kThreads;
using paged::kWarps;
using paged::ldsm4;
using paged::ldsm4t;
using paged::log2_of;
using paged::mma;
using paged::pack2;
using paged::rotate;
using paged::Shares;
using paged::unpack2;

__device__ int g_err;

constexpr int kRows = 16;                  // slots of a tile, an MMA's rows
constexpr int kPair = 2 * kRows;           // slots of a stage: two tiles
constexpr int kUnit = kWarps * kPair;      // slots of a unit
constexpr float kSlack = 4.f;              // log2 by which a weight may pass 1 before the maximum follows
constexpr float kShift = 11.f;             // weights are 2^kShift times: at most 2^15, in fp16 down to 2^-35 times

struct AttnArgs {
  Cache c;
  const uint16_t* q;
  int64_t q_stride;
  int n_q, group, head_tiles;
  int abreast;           // rows of a sequence that CTAs of neighbouring numbers take side by side
  int extra;             // 1: slot seq_lens[b] holds the new token and counts
  const int64_t* positions;
  const float* cos_t;
  const float* sin_t;
  int64_t rope_rows;
  float scale2;          // scale * log2(e)
  uint16_t* out;
  int64_t out_stride;
  int* counters;
  float* partials;       // [grid][2][heads of a tile][D + 2]: the heads' rows, each with its max and sum
  int page_shift;        // log2(page_size), or -1
  int whole_pairs;       // page_size % 32 == 0: both tiles of a stage share a page
  uint64_t wait_ns;
  int stall;             // test hook: nothing is loaded
};

// Slots that sequence b attends over: 0 without any, or without a place for the new token.
__device__ __forceinline__ int slots_of(const AttnArgs& a, int len) {
  if (len < 0 || len > (int64_t)a.c.max_pages * a.c.page_size - a.extra) return 0;
  return len + a.extra;
}
__device__ __forceinline__ int units_of(const AttnArgs& a, int len) { return (slots_of(a, len) + kUnit - 1) / kUnit; }

__device__ __forceinline__ int page_index(const AttnArgs& a, int slot) {
  return a.page_shift >= 0 ? slot >> a.page_shift : slot / a.c.page_size;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int s, int h, int p, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(s), "r"(h), "r"(p), "r"(smem_u32(bar))
      : "memory");
}

// The 8 x 8 matrix of fp16 pairs that a warp holds, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t w) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(w));
  return d;
}

// Four codes as fp16: x of bytes 0, 1 and y of bytes 2, 3, or (SPLIT) x of 0, 2 and y of 1, 3.
template <bool E4M3, bool SPLIT>
__device__ __forceinline__ void to_half(uint32_t w, uint32_t& x, uint32_t& y) {
  if constexpr (E4M3) {
    if (SPLIT) w = prmt(w, 0, 0x3120);
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
        : "=r"(x), "=r"(y) : "r"(w));
  } else {
    // 1024 + (code + 128) as fp16, whose lowest mantissa bit stands for 1
    w ^= 0x80808080u;
    const uint32_t magic = 0x64646464u;
    x = prmt(w, magic, SPLIT ? 0x4240 : 0x4140);
    y = prmt(w, magic, SPLIT ? 0x4341 : 0x4342);
    asm("sub.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0x64806480u));   // 1152
    asm("sub.f16x2 %0, %0, %1;" : "+r"(y) : "r"(0x64806480u));
  }
}

// Shared memory of a block: the warps' rings [kWarps][S][K, V][boxes][32 rows][kBox], their
// barriers, the query tile ([heads][DP + 8] fp16, or three planes of bytes [heads][DP + 16]),
// the heads' powers of two, and the prefix sums of the sequences' units with their lengths.
//
// DP: columns that are computed, head_dim rounded up (the copies fill the rest of a
// box with zeros). C: blocks per SM, as many as the registers allow, which hides more of a
// tile's chain of latencies, and of a row's start, than longer rings do. 64 columns, 64 sequences
// of up to 16000 slots: four blocks 108 us, three 112, two with rings of six stages 139;
// 16 query heads to a kv head, 32 of up to 8000: 54, 53, 57. 96 columns, 64 of up to
// 16000: three blocks 141, two 156; 128 columns: see kManyRows.
template <int DP, int NT, int C>
struct Ring {
  static constexpr int kCols = DP <= 64 ? 64 : DP <= 128 ? 128 : 256;   // columns in shared memory
  static constexpr int kBox = kCols < 128 ? kCols : 128;        // columns of a TMA box
  static constexpr int kHalf = kPair * kCols;                   // bytes of a stage's K (or V)
  static constexpr int kStage = 2 * kHalf;
  static constexpr int S = kCols == 128 && C == 3 ? 2 : 3;
  static constexpr size_t kBytes = (size_t)kWarps * S * kStage;
};

// 128 columns: three blocks per SM with rings of two stages where the rows are many and short (150
// sequences of 8 kv heads, of up to 300 slots 30 us for 33 with two blocks of three stages, of
// up to 3000 91 for 103), else two (128 of 8000 slots 328 us for 337, 64 of up to 16000 175 for
// 176, 4 of 4000 17.9 for 18.9). The host knows the tables' capacity, not the lengths: 256 of up to 1000 slots
// in tables with room for more than 4096 take 81 us, 68 with three blocks.
constexpr int kManyRows = 2;               // kv heads of all sequences per SM, from which three are taken
constexpr int64_t kShortTable = 4096;      // slots

template <bool E4M3, int DP, int NT>
constexpr bool int_scores() { return !E4M3 && DP * NT <= 128; }
template <bool E4M3, int DP, int NT>
constexpr size_t q_bytes() { return int_scores<E4M3, DP, NT>() ? 3 * 8 * NT * (DP + 16) : 8 * NT * (DP + 8) * 2; }
template <bool E4M3, int DP, int NT, int C>
constexpr size_t attn_smem(int batch) {
  return 1024 + Ring<DP, NT, C>::kBytes + kWarps * Ring<DP, NT, C>::S * 8 + q_bytes<E4M3, DP, NT>() + 8 * NT * 4 +
         (size_t)(2 * batch + 1) * 4;
}

// 16 x 8 sums of 32 products of bytes.
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool BF, bool E4M3, int DP, int NT, int C>
__global__ void __launch_bounds__(kThreads, C)
    paged8_attention_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const AttnArgs a) {
  using P = Ring<DP, NT, C>;
  constexpr bool kInt = int_scores<E4M3, DP, NT>();
  constexpr int S = P::S;
  constexpr int kHeads = 8 * NT;                 // query heads of a tile: a multiple of kWarps
  constexpr int kBlocks = DP / 16;               // steps of 16 columns
  constexpr int kQPitch = DP + 8;
  extern __shared__ char smem_raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + P::kBytes);                       // [kWarps][S]
  uint16_t* qs = reinterpret_cast<uint16_t*>(bars + kWarps * S);                        // [kHeads][kQPitch]
  char* q8 = reinterpret_cast<char*>(qs);                                               // [3][kHeads][DP + 16]
  float* q_pow = reinterpret_cast<float*>(q8 + q_bytes<E4M3, DP, NT>());                // [kHeads]
  int* prefix = reinterpret_cast<int*>(q_pow + kHeads);                                 // [batch + 1]
  __shared__ uint64_t warp_sums[kWarps];
  __shared__ int warp_most[kWarps];
  __shared__ int is_last;
  const Cache& c = a.c;
  int* lens = prefix + c.batch + 1;                                                     // [batch]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int D = c.head_dim, rows_per_b = c.n_kv * a.head_tiles;
  const int laid = rows_per_b / a.abreast;               // rows of a sequence that lie end to end
  // CTAs abreast work as one on the rows laid end to end, each on a row of its own of every `abreast`
  const unsigned cta = blockIdx.x / a.abreast, side = blockIdx.x - cta * a.abreast;

  if (tid == 0) {
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
    for (int i = 0; i < kWarps * S; ++i) mbar_init(bars + i, 1);
    fence_barrier_init();
  }
  // prefix sums of the sequences' units; every thread takes a run of sequences
  int longest = 0;
  Deal deal;
  {
    const int per = (c.batch + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, c.batch), b1 = min(b0 + per, c.batch);
    uint64_t sum = 0;                             // units, and sequences with units in the upper half
    int most = 0;
    for (int b = b0; b < b1; ++b) {
      lens[b] = c.seq_lens[b];
      const int n = units_of(a, lens[b]);
      sum += n > 0 ? ((uint64_t)1 << 32) + n : 0;
      most = max(most, n);
    }
    uint64_t inc = sum;
    most = __reduce_max_sync(0xffffffffu, most);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    if (lane == 31) {
      warp_sums[warp] = inc;
      warp_most[warp] = most;
    }
    __syncthreads();
    uint64_t all = 0, at = inc - sum;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      longest = max(longest, warp_most[w]);
      if (w < warp) at += warp_sums[w];
      all += warp_sums[w];
    }
    // How the units are dealt out: a row of n units counts n + front, or, with
    // front < 0, -front whatever n is.
    const unsigned units = (unsigned)(uint32_t)all * laid, rows = (unsigned)(all >> 32) * laid;
    deal = choose_deal(units, rows, longest, gridDim.x / a.abreast, min(a.group, kHeads));
    int v = 0;
    if (deal.front >= 0) v = (int)(uint32_t)at + deal.front * (int)(at >> 32);
    else v = -deal.front * (int)(at >> 32);
    for (int b = b0; b < b1; ++b) {
      prefix[b] = v;
      const int n = units_of(a, lens[b]);
      v += n > 0 ? (deal.front >= 0 ? n + deal.front : -deal.front) : 0;
    }
    if (b1 == c.batch && b0 < b1) prefix[c.batch] = v;
  }
  // query columns and heads that nothing fills: zeros, so that their scores are finite
  for (int i = tid; i < (int)q_bytes<E4M3, DP, NT>() / 4; i += kThreads) reinterpret_cast<uint32_t*>(qs)[i] = 0;
  if (tid < kHeads) q_pow[tid] = 0.f;
  __syncthreads();
  pdl_wait_primary();                                    // (the kernel that stores the new token)
  // a sequence without slots answers with zeros
  for (int b = blockIdx.x; b < c.batch; b += gridDim.x)
    if (prefix[b] == prefix[b + 1])
      for (int i = tid; i < a.n_q * D; i += kThreads) a.out[b * a.out_stride + i] = 0;

  const unsigned total = (unsigned)prefix[c.batch] * laid;         // (the host keeps it below 2^31)
  if (total == 0) return;
  const unsigned n_cta = min(deal.n_cta, total);
  if (cta >= n_cta) return;
  const Shares shares(total, n_cta);
  const unsigned u1 = shares.begin(cta + 1);

  char* ring = smem + (size_t)warp * S * P::kStage;
  const uint32_t ring_u = smem_u32(ring);
  uint64_t* bar = bars + warp * S;
  uint32_t phases = 0;                                   // a bit per stage: the parity of its next completion
  bool broken = false;

  // the first row: sequence b is the last with prefix[b] * laid <= u
  unsigned u = shares.begin(cta);
  int b = 0;
  for (int hi = c.batch - 1; b < hi;) {
    const int mid = (b + hi + 1) >> 1;
    if ((unsigned)prefix[mid] * laid <= u) b = mid; else hi = mid - 1;
  }
  int nth = (int)((u - (unsigned)prefix[b] * laid) / (unsigned)(prefix[b + 1] - prefix[b]));
  for (; u < u1; ++nth) {
    // the segment: units [t0, t1) of (sequence b, kv head h, head tile ht)
    if (nth == laid) {
      nth = 0;
      do ++b; while (prefix[b + 1] == prefix[b]);
    }
    const int cost = prefix[b + 1] - prefix[b], nt = units_of(a, lens[b]), front = cost - nt;
    const unsigned row_u = (unsigned)prefix[b] * laid + (unsigned)(nth * cost);
    const int v0 = (int)(u - row_u), v1 = (int)min((unsigned)cost, v0 + (u1 - u));
    u += v1 - v0;
    if (v1 <= front) continue;                         // only the row's front
    const int t0 = max(v0 - front, 0), t1 = v1 - front;
    const int row = nth * a.abreast + (int)side;
    const int h = row / a.head_tiles, ht = row - h * a.head_tiles;
    const int heads = min(kHeads, a.group - ht * kHeads);
    const int head0 = h * a.group + ht * kHeads;       // first query head of the tile
    const int n = slots_of(a, lens[b]);
    const int32_t* table = c.table + b * c.table_stride;

    // Stage k of this warp: slots t0 * 128 + warp * 32 + 128 k on, tiles 2 k and 2 k + 1. Lane i
    // holds page and scales of tile i of the current batch of 32 (pg, ka, va) and of
    // the next one (pg1, ...), and the pages of the one after that.
    const int slot_base = t0 * kUnit + warp * kPair;
    const int stages = min(t1 - t0, (n - slot_base + kUnit - 1) / kUnit);
    auto slot_of_tile = [&](int j) { return slot_base + (j >> 1) * kUnit + (j & 1) * kRows; };
    auto page_of_tile = [&](int j) {
      const int slot = slot_of_tile(j);
      const int p = j < 2 * stages && slot < n ? table[page_index(a, slot)] : -1;
      return (unsigned)p < (unsigned)c.num_pages ? p : -1;
    };
    auto scales_of_tile = [&](int j, int page, float& ka, float& va) {
      ka = va = 0.f;
      if (page >= 0) {
        const int slot = slot_of_tile(j);
        const int64_t at = scale_at(c, page, h, (slot - page_index(a, slot) * c.page_size) / c.block);
        ka = c.k_scales[at];
        va = c.v_scales[at];
      }
    };
    int pg = page_of_tile(lane), pg1 = page_of_tile(32 + lane), pg2;
    float ka, va, ka1, va1;

    // What the segment needs first is loaded before the copies, behind which it would wait: the
    // position, the rotation, the query heads (each by a warp: elements j and j + D / 2).
    const bool turn = a.cos_t != nullptr;
    const int64_t pos_in = a.positions != nullptr ? a.positions[b] : lens[b];
    constexpr int kPer = (DP / 2 + 31) / 32, kOwn = kHeads / kWarps;
    uint32_t qx[kOwn][kPer];
#pragma unroll
    for (int w = 0; w < kOwn; ++w) {
      const int g = warp + w * kWarps;
      const uint16_t* qr = a.q + b * a.q_stride + (int64_t)(head0 + g) * D;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int j = lane + 32 * i;
        qx[w][i] = g < heads && j < D / 2 ? (uint32_t)qr[j] | ((uint32_t)qr[j + D / 2] << 16) : 0;
      }
    }
    bool ok = !turn || (pos_in >= 0 && pos_in < a.rope_rows);
    if (a.extra) {
      // (a new token without a page answers with zeros)
      const int p = table[page_index(a, lens[b])];
      ok = ok && (unsigned)p < (unsigned)c.num_pages;
    }
    float2 rot[kPer];
    if (turn) {
      const int64_t at = (ok ? pos_in : 0) * (D / 2);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int j = min(lane + 32 * i, D / 2 - 1);
        rot[i] = make_float2(a.cos_t[at + j], a.sin_t[at + j]);
      }
    }
    scales_of_tile(lane, pg, ka, va);

    // Copies stage k to place `at` of the ring, tiles with a page; their bytes complete on its barrier.
    auto issue = [&](int k, int at, int page0, int page1) {
      if ((page0 < 0 && page1 < 0) || a.stall || broken) return;
      if (elect_one()) {
        const int slot = slot_of_tile(2 * k), i = page_index(a, slot), off = slot - i * c.page_size;
        const uint32_t dst = ring_u + at * P::kStage;
        if (a.whole_pairs) {                             // both tiles lie in one page
          mbar_arrive_expect_tx(bar + at, P::kStage);
#pragma unroll
          for (int x = 0; x < P::kCols / P::kBox; ++x) {
            tma_load_4d(dst + x * kPair * P::kBox, &kmap, x * P::kBox, off, h, page0, bar + at);
            tma_load_4d(dst + P::kHalf + x * kPair * P::kBox, &vmap, x * P::kBox, off, h, page0, bar + at);
          }
        } else {
          mbar_arrive_expect_tx(bar + at, (page0 >= 0 && page1 >= 0 ? 1 : 0) * (P::kStage / 2) + P::kStage / 2);
          const int off1 = off + kRows < c.page_size ? off + kRows : 0;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int page = e == 0 ? page0 : page1, o = e == 0 ? off : off1;
            if (page < 0) continue;
#pragma unroll
            for (int x = 0; x < P::kCols / P::kBox; ++x) {
              const uint32_t d = dst + (x * kPair + e * kRows) * P::kBox;
              tma_load_4d(d, &kmap, x * P::kBox, o, h, page, bar + at);
              tma_load_4d(d + P::kHalf, &vmap, x * P::kBox, o, h, page, bar + at);
            }
          }
        }
      }
      __syncwarp();
    };
#pragma unroll
    for (int k = 0; k < S; ++k)
      issue(k, k, __shfl_sync(0xffffffffu, pg, 2 * k), __shfl_sync(0xffffffffu, pg, 2 * k + 1));
    scales_of_tile(32 + lane, pg1, ka1, va1);
    pg2 = page_of_tile(64 + lane);

    // Each head by a warp: rotated and rounded to its type, then either in fp16 with the
    // power of two of its largest magnitude taken out (off by 2^-25 of that power at most, where an
    // element lies under fp16's normal range, else not at all), or as an integer of 2^21
    // times that, in three signed bytes (24 bits under the largest magnitude, off by 2^-22 of the power at most).
#pragma unroll
    for (int w = 0; w < kOwn; ++w) {
      const int g = warp + w * kWarps;
      if (g >= heads) break;
      uint32_t* x = qx[w];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (turn) {
          const float2 f = unpack2<BF>(x[i]);
          const float2 y = rotate(f.x, f.y, rot[i].x, rot[i].y);
          x[i] = lane + 32 * i < D / 2 ? pack2<BF>(y.x, y.y) : 0;
        }
        top = __vmaxu2(top, x[i] & 0x7FFF7FFFu);
      }
      top = __reduce_max_sync(0xffffffffu, max(top & 0xFFFFu, top >> 16));
      const uint32_t e = min(max(__float_as_uint(unpack2<BF>(top).x) >> 23, 20u), 253u);
      const float down = __uint_as_float((254u - e) << 23);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int j = lane + 32 * i;
        if (j < D / 2) {
          const float2 f = unpack2<BF>(x[i]);
          if constexpr (kInt) {
            auto put = [&](float y, int at) {
              const int v = max(-8355711, min(8355711, __float2int_rn(y * down * 2097152.f)));   // (the largest three bytes)
              const int b0 = (int8_t)v, v1 = (v - b0) >> 8, b1 = (int8_t)v1;
              char* p = q8 + g * (DP + 16) + at;
              p[0] = (char)b0;
              p[kHeads * (DP + 16)] = (char)b1;
              p[2 * kHeads * (DP + 16)] = (char)((v1 - b1) >> 8);
            };
            put(f.x, j);
            put(f.y, j + D / 2);
          } else {
            const uint32_t w = pack2<false>(f.x * down, f.y * down);
            qs[g * kQPitch + j] = (uint16_t)w;
            qs[g * kQPitch + j + D / 2] = (uint16_t)(w >> 16);
          }
        }
      }
      // (a head with an infinity or a NaN has no scores)
      const float unit = kInt ? 4.76837158203125e-7f : 1.f;     // 2^-21
      if (lane == 0) q_pow[g] = top < (BF ? 0x7F80u : 0x7C00u) ? __uint_as_float(e << 23) * unit : __uint_as_float(0x7FC00000u);
    }
    __syncthreads();
    // operand registers of q, of head lane / 4: columns 4 i .. 4 i + 3 of every 16 (fp16); or 4 i .. and
    // 16 + 4 i .. of every 32, for each plane of bytes
    uint2 qf[kInt ? 3 * kBlocks / 2 : kBlocks][NT];
    float f[NT][2];                                    // scale and power of two of this thread's heads
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if constexpr (kInt) {
#pragma unroll
        for (int p = 0; p < 3; ++p)
#pragma unroll
          for (int s = 0; s < kBlocks / 2; ++s) {
            const char* src = q8 + (p * kHeads + 8 * t + (lane >> 2)) * (DP + 16) + 32 * s + 4 * (lane & 3);
            qf[p * (kBlocks / 2) + s][t] =
                make_uint2(*reinterpret_cast<const uint32_t*>(src), *reinterpret_cast<const uint32_t*>(src + 16));
          }
      } else {
#pragma unroll
        for (int s = 0; s < kBlocks; ++s)
          qf[s][t] = *reinterpret_cast<const uint2*>(qs + (8 * t + (lane >> 2)) * kQPitch + 16 * s + 4 * (lane & 3));
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) f[t][e] = q_pow[8 * t + 2 * (lane & 3) + e] * a.scale2;
    }

    // o[s][t]: columns 16 s + 2 g (first two) and + 1 of heads 8 t + 2 i and + 1, g = lane / 4, i = lane % 4
    float o[kBlocks][NT][4];
#pragma unroll
    for (int s = 0; s < kBlocks; ++s)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[s][t][e] = 0.f;
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
    }
    float v_pow = 0.f, v_inv = 0.f;                    // the power of two over the values' scales, and its inverse

    const int g8 = lane >> 2;
    // Byte (row r, column d) of a box: 16-byte chunk d / 16 is kept at another place of its row,
    // its number xor r % 8 (of rows of 64 bytes: r / 2 % 4), so that eight rows of a chunk
    // touch every bank once. This lane's row and chunk of an ldmatrix, whose matrices are (slots 0-7,
    // chunk 2 s), (8-15, 2 s), (0-7, 2 s + 1), (8-15, 2 s + 1):
    const uint32_t l_at = (lane & 15) * P::kBox + (((lane >> 4) ^ (P::kBox == 128 ? lane & 7 : (lane >> 1) & 3)) << 4);
    auto chunks_at = [&](uint32_t base, int s) {       // (tiles start on multiples of their size)
      return ((base + l_at) ^ ((s << 5) % P::kBox)) + (s << 5) / P::kBox * (kPair * P::kBox);
    };

    // Waits for the stage at `at`; false if that took too long.
    auto arrived = [&](int at) {
      if (!__all_sync(0xffffffffu, mbar_wait_hint(bar + at, (phases >> at) & 1, &g_err, 61, a.wait_ns))) return false;
      phases ^= 1u << at;
      return true;
    };

    // Takes the tile at byte `at` of the ring, whose block has the scales ks, vs and whose first
    // `live` slots count.
    auto consume = [&](int at, float ks, float vs, int live) {
      const uint32_t kb = ring_u + at, vb = kb + P::kHalf;
      if (live < kRows) {
        // values behind the last token may be anything, an e4m3 NaN too, which no weight of 0 hides
        char* v = ring + at + P::kHalf;
        for (int x = lane; x < (kRows - live) * (P::kCols / 16); x += 32) {
          const int r = live + x / (P::kCols / 16), ch = x % (P::kCols / 16);
          *reinterpret_cast<uint4*>(v + (ch * 16 / P::kBox) * kPair * P::kBox + r * P::kBox + (ch * 16 % P::kBox)) =
              make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      float sc[NT][4];                                 // scores of 16 slots x the tile's heads
      if constexpr (kInt) {
        int si[NT][3][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int p = 0; p < 3; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e) si[t][p][e] = 0;
#pragma unroll
        for (int s = 0; s < kBlocks / 2; ++s) {
          uint32_t w[4];
          ldsm4(chunks_at(kb, s), w);
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int p = 0; p < 3; ++p) mma_s8(si[t][p], w, qf[p * (kBlocks / 2) + s][t].x, qf[p * (kBlocks / 2) + s][t].y);
        }
        // (the lower two planes together stay below 2^31)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[t][e] = fmaf((float)si[t][2][e], 65536.f, (float)(si[t][1][e] * 256 + si[t][0][e]));
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[t][e] = 0.f;
#pragma unroll
        for (int s = 0; s < kBlocks / 2; ++s) {
          uint32_t w[4];
          ldsm4(chunks_at(kb, s), w);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t k4[4];
            to_half<E4M3, false>(w[2 * e], k4[0], k4[2]);
            to_half<E4M3, false>(w[2 * e + 1], k4[1], k4[3]);
#pragma unroll
            for (int t = 0; t < NT; ++t) mma<false>(sc[t], k4, qf[2 * s + e][t].x, qf[2 * s + e][t].y);
          }
        }
      }
      // in log2 units
      bool past = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float f0 = f[t][0] * ks, f1 = f[t][1] * ks;
        sc[t][0] *= f0;
        sc[t][1] *= f1;
        sc[t][2] *= f0;
        sc[t][3] *= f1;
        if (live < kRows) {
          if (g8 >= live) sc[t][0] = sc[t][1] = -INFINITY;
          if (g8 + 8 >= live) sc[t][2] = sc[t][3] = -INFINITY;
        }
        past = past || fmaxf(sc[t][0], sc[t][2]) > m[t][0] + kSlack || fmaxf(sc[t][1], sc[t][3]) > m[t][1] + kSlack;
      }
      if (__any_sync(0xffffffffu, past || fabsf(vs) > v_pow)) {
        float grow = 1.f;
        if (fabsf(vs) > v_pow) {
          const uint32_t e = min((__float_as_uint(fabsf(vs)) + 0x7FFFFFu) >> 23, 253u);     // 2^e >= |vs|
          const float inv = __uint_as_float((254u - e) << 23);
          grow = v_pow * inv;
          v_pow = __uint_as_float(e << 23);
          v_inv = inv;
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(sc[t][e], sc[t][e + 2]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const float mn = fmaxf(m[t][e], x);
            const float corr = mn == -INFINITY ? 1.f : ex2(m[t][e] - mn);
            m[t][e] = mn;
            l[t][e] *= corr;
            const float both = corr * grow;
#pragma unroll
            for (int s = 0; s < kBlocks; ++s) {
              o[s][t][e] *= both;
              o[s][t][e + 2] *= both;
            }
          }
      }
      const float vf = vs * v_inv;                     // 1 in size at most
      uint32_t pf[NT][2], pr[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        // (a maximum of -inf: no score was a number, and the weights become NaN or 0)
        const float m0 = m[t][0] == -INFINITY ? 0.f : m[t][0] - kShift, m1 = m[t][1] == -INFINITY ? 0.f : m[t][1] - kShift;
        float p[4] = {ex2(sc[t][0] - m0), ex2(sc[t][1] - m1), ex2(sc[t][2] - m0), ex2(sc[t][3] - m1)};
        l[t][0] += p[0] + p[2];
        l[t][1] += p[1] + p[3];
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] *= vf;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t w = pack2<false>(p[2 * e], p[2 * e + 1]);
          const float2 x = unpack2<false>(w);
          pf[t][e] = transpose8(w);
          pr[t][e] = transpose8(pack2<false>(p[2 * e] - x.x, p[2 * e + 1] - x.y));
        }
      }
#pragma unroll
      for (int s = 0; s < kBlocks / 2; ++s) {
        uint32_t w[4];
        ldsm4t(chunks_at(vb, s), w);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t v4[4];
          to_half<E4M3, true>(w[2 * e], v4[0], v4[1]);
          to_half<E4M3, true>(w[2 * e + 1], v4[2], v4[3]);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma<false>(o[2 * s + e][t], v4, pf[t][0], pf[t][1]);
            mma<false>(o[2 * s + e][t], v4, pr[t][0], pr[t][1]);
          }
        }
      }
    };

    int place = 0;
    for (int k = 0; k < stages && !broken; ++k) {
      const int i = 2 * k & 31;                        // of the batch
      if (i == 0 && k > 0) {
        pg = pg1; ka = ka1; va = va1;
        pg1 = pg2;
        scales_of_tile(2 * k + 32 + lane, pg1, ka1, va1);
        pg2 = page_of_tile(2 * k + 64 + lane);
      }
      const int page[2] = {__shfl_sync(0xffffffffu, pg, i), __shfl_sync(0xffffffffu, pg, i + 1)};   // (-1: nothing was loaded)
      const float ks[2] = {__shfl_sync(0xffffffffu, ka, i), __shfl_sync(0xffffffffu, ka, i + 1)};
      const float vs[2] = {__shfl_sync(0xffffffffu, va, i), __shfl_sync(0xffffffffu, va, i + 1)};
      if (page[0] >= 0 || page[1] >= 0) {
        if (!arrived(place)) {
          broken = true;
          // the copies that are on their way land before the block ends
          if (!a.stall)
            for (int e = 0; e < S; ++e) {
              const int x = i + 2 * e, st = (place + e) % S;
              const int p0 = __shfl_sync(0xffffffffu, x < 32 ? pg : pg1, x & 31), p1 = __shfl_sync(0xffffffffu, x < 32 ? pg : pg1, (x + 1) & 31);
              if (k + e < stages && (p0 >= 0 || p1 >= 0)) mbar_wait_hint(bar + st, (phases >> st) & 1, nullptr, 0, a.wait_ns);
            }
          break;
        }
#pragma unroll 1
        for (int e = 0; e < 2; ++e)
          if ((e == 0 ? page[0] : page[1]) >= 0)
            consume(place * P::kStage + e * kRows * P::kBox, e == 0 ? ks[0] : ks[1], e == 0 ? vs[0] : vs[1],
                    n - slot_of_tile(2 * k + e));
        __syncwarp();
      }
      {
        const int x = i + 2 * S;
        issue(k + S, place, __shfl_sync(0xffffffffu, x < 32 ? pg : pg1, x & 31),
              __shfl_sync(0xffffffffu, x < 32 ? pg : pg1, (x + 1) & 31));
      }
      place = place + 1 == S ? 0 : place + 1;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 4);
        l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 8);
        l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 16);
      }
    __syncthreads();

    // join the warps through shared memory (over the drained rings)
    constexpr int kJoin = DP + 4;                    // floats of a row: its sums, max, sum
    float* jo = reinterpret_cast<float*>(smem);      // [kWarps][kHeads][kJoin]
    static_assert((size_t)kWarps * kHeads * (kJoin + 2) * 4 + 64 <= P::kBytes, "join area");
    const float v_fin = v_pow * exp2f(-kShift), l_fin = exp2f(-kShift);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float* r = jo + (warp * kHeads + 8 * t + 2 * (lane & 3) + e) * kJoin;
#pragma unroll
        for (int s = 0; s < kBlocks; ++s)
          *reinterpret_cast<float2*>(r + 16 * s + 2 * g8) = make_float2(o[s][t][e] * v_fin, o[s][t][e + 2] * v_fin);
        if (g8 == 0) {
          r[DP] = m[t][e];
          r[DP + 1] = l[t][e] * l_fin;
        }
      }
    __syncthreads();
    // factors 2^(m_warp - m) of every warp and head, then the sums
    float* fac = jo + kWarps * kHeads * kJoin;       // [kWarps][kHeads], then [kHeads] maxima, [kHeads] sums
    if (tid < kHeads) {
      float wm[kWarps], mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, wm[w] = jo[(w * kHeads + tid) * kJoin + DP]);
      const float bs = mm == -INFINITY ? 0.f : mm;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float y = ex2(wm[w] - bs);
        fac[w * kHeads + tid] = y;
        ll = fmaf(y, jo[(w * kHeads + tid) * kJoin + DP + 1], ll);
      }
      fac[kWarps * kHeads + tid] = mm;
      fac[(kWarps + 1) * kHeads + tid] = ll;
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == nt;
    const int64_t prow = (int64_t)kHeads * (D + 2);  // a piece: [kHeads][D] sums, [kHeads] (max, sum)
    // a CTA has at most two partial rows: one that it ends, one that it begins
    float* part = a.partials + ((int64_t)blockIdx.x * 2 + (t0 > 0 ? 0 : 1)) * prow;
    uint16_t* out = a.out + b * a.out_stride + (int64_t)head0 * D;
    for (int i = tid; i < heads * (D / 4); i += kThreads) {
      const int g = i / (D / 4), d = 4 * (i - g * (D / 4));
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(jo + (w * kHeads + g) * kJoin + d);
        const float y = fac[w * kHeads + g];
        acc.x = fmaf(y, v.x, acc.x);
        acc.y = fmaf(y, v.y, acc.y);
        acc.z = fmaf(y, v.z, acc.z);
        acc.w = fmaf(y, v.w, acc.w);
      }
      if (whole) {
        // (no slot with a page: zeros)
        const float ll = fac[(kWarps + 1) * kHeads + g], inv = ll == 0.f ? 0.f : 1.f / ll;
        uint32_t* dst = reinterpret_cast<uint32_t*>(out + g * D + d);
        dst[0] = ok ? pack2<BF>(acc.x * inv, acc.y * inv) : 0;
        dst[1] = ok ? pack2<BF>(acc.z * inv, acc.w * inv) : 0;
      } else {
        *reinterpret_cast<float4*>(part + g * D + d) = acc;
      }
    }
    if (tid < heads && !whole)
      reinterpret_cast<float2*>(part + kHeads * D)[tid] = make_float2(fac[kWarps * kHeads + tid], fac[(kWarps + 1) * kHeads + tid]);
    if (!whole) {
      const unsigned first_u = row_u + front;        // the row's first unit
      const int cta0 = (int)shares.owner(first_u), cta1 = (int)shares.owner(first_u + nt - 1);
      int* cnt = a.counters + b * rows_per_b + row;
      __syncthreads();
      if (tid == 0) {
        // releases the CTA's piece (ordered before by the barrier) and acquires
        // the others'
        int seen;
        asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(seen) : "l"(cnt) : "memory");
        is_last = seen == cta1 - cta0;
        if (is_last) *cnt = 0;                       // zero for the next call
      }
      __syncthreads();
      if (is_last) {
        const int pieces = cta1 - cta0 + 1;          // at most kMaxPieces + 1
        // a row's pieces lie first in their CTAs' slots, but for its beginning
        const float* others = a.partials + ((int64_t)cta0 * a.abreast + side) * 2 * prow;
        const int64_t next = (int64_t)a.abreast * 2 * prow;
        auto piece = [&](int i) { return i == 0 ? others + prow : others + i * next; };
        // Two heads per warp, which needs no other: the pieces' factors
        // 2^(m_piece - m), lane i those of pieces i, i + 32, ..., and their sums, four
        // values a lane, eight pieces in flight ahead of their use.
        constexpr int kML = (kMaxPieces + 1 + 31) / 32, kAhead = 8;
        for (int g0 = warp; g0 < heads; g0 += 2 * kWarps) {
          const int second = g0 + kWarps < heads ? kWarps * D : 0;   // (an odd head is summed twice)
          float4 v[kAhead][2];
          auto load = [&](int i0, int d) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
              const float* src = piece(min(i0 + i, pieces - 1)) + g0 * D + (d < D ? d : 0);
              v[i][0] = __ldcg(reinterpret_cast<const float4*>(src));
              v[i][1] = __ldcg(reinterpret_cast<const float4*>(src + second));
            }
          };
          load(0, 4 * lane);
          float y[2][kML], inv[2];
          {
            float2 ml[2][kML];
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
              for (int k = 0; k < kML; ++k) {
                const int i = lane + 32 * k, g = g0 + e * kWarps;
                ml[e][k] = i < pieces && g < heads ? __ldcg(reinterpret_cast<const float2*>(piece(i) + kHeads * D) + g)
                                                   : make_float2(-INFINITY, 0.f);
              }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mm = -INFINITY, ll = 0.f;
#pragma unroll
              for (int k = 0; k < kML; ++k) mm = fmaxf(mm, ml[e][k].x);
#pragma unroll
              for (int o2 = 16; o2 > 0; o2 >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o2));
              const float bs = mm == -INFINITY ? 0.f : mm;
#pragma unroll
              for (int k = 0; k < kML; ++k) {
                y[e][k] = ex2(ml[e][k].x - bs);
                ll = fmaf(y[e][k], ml[e][k].y, ll);
              }
              ll = warp_sum(ll);
              inv[e] = ll == 0.f ? 0.f : 1.f / ll;
            }
          }
          for (int d = 4 * lane; d - 4 * lane < D; d += 128) {
            if (d != 4 * lane) load(0, d);
            float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
            for (int i0 = 0; i0 < pieces; i0 += kAhead) {
#pragma unroll
              for (int i = 0; i < kAhead; ++i) {
                if (i0 + i >= pieces) break;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  // the factor of piece i0 + i
                  float w = y[e][0];
#pragma unroll
                  for (int k = 1; k < kML; ++k) w = i0 >= 32 * k ? y[e][k] : w;
                  w = __shfl_sync(0xffffffffu, w, (i0 + i) & 31);
                  acc[e].x = fmaf(w, v[i][e].x, acc[e].x);
                  acc[e].y = fmaf(w, v[i][e].y, acc[e].y);
                  acc[e].z = fmaf(w, v[i][e].z, acc[e].z);
                  acc[e].w = fmaf(w, v[i][e].w, acc[e].w);
                }
              }
              if (i0 + kAhead < pieces) load(i0 + kAhead, d);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (d >= D || (e == 1 && second == 0)) continue;
              uint32_t* dst = reinterpret_cast<uint32_t*>(out + (g0 + e * kWarps) * D + d);
              dst[0] = ok ? pack2<BF>(acc[e].x * inv[e], acc[e].y * inv[e]) : 0;
              dst[1] = ok ? pack2<BF>(acc[e].z * inv[e], acc[e].w * inv[e]) : 0;
            }
          }
        }
      }
    }
    fence_proxy_async_smem();   // the join area becomes the rings again, which copies write
    __syncthreads();
  }
}

static size_t workspace_bytes_of(int head_dim) {
  const int ctas = head_dim > 128 ? 1 : head_dim > 64 ? 3 : 4;   // blocks per SM at most
  return kCounterBytes + (size_t)sm_count() * ctas * 2 * 16 * (head_dim + 2) * 4;
}

static int encode_map(CUtensorMap* map, const Cache& c, const void* base, int box) {
  const uint64_t dims[4] = {(uint64_t)c.head_dim, (uint64_t)c.page_size, (uint64_t)c.n_kv, (uint64_t)c.num_pages};
  // (of a dimension of one the stride does not matter, but it has to be a valid one)
  auto stride = [&](int64_t s, int n) { return (uint64_t)(n > 1 ? s : std::max<int64_t>(s, 16)); };
  const uint64_t strides[3] = {stride(c.token_stride, c.page_size), stride(c.head_stride, c.n_kv), stride(c.page_stride, c.num_pages)};
  const uint32_t boxes[4] = {(uint32_t)box, (uint32_t)(c.page_size % kPair == 0 ? kPair : kRows), 1, 1};
  return encode_tmap(map, base, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, dims, strides, boxes,
                     box == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
}

// `token`: what is appended first, once nothing can be refused any more; or NULL.
template <bool BF, bool E4M3, int DP, int NT, int C>
static int launch(const AttnArgs& a, const AppendArgs* token, cudaStream_t st) {
  auto k = paged8_attention_kernel<BF, E4M3, DP, NT, C>;
  const size_t smem = attn_smem<E4M3, DP, NT, C>(a.c.batch);
  // (the same value for all host threads, as for the 16-bit kernel)
  static thread_local int configured_dev = -1;
  static thread_local size_t most = 0;
  int dev = 0;
  TS_CUDA_TRY(cudaGetDevice(&dev));
  if (configured_dev != dev) {
    cudaFuncAttributes attr;
    TS_CUDA_TRY(cudaFuncGetAttributes(&attr, k));
    most = (size_t)max_smem_optin() - attr.sharedSizeBytes;
    TS_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    configured_dev = dev;
  }
  TS_UNSUPPORTED(smem <= most, "batch too large for the kernel's tables");
  CUtensorMap km, vm;
  int rc = encode_map(&km, a.c, a.c.k, Ring<DP, NT, C>::kBox);
  if (rc == TS_OK) rc = encode_map(&vm, a.c, a.c.v, Ring<DP, NT, C>::kBox);
  if (rc == TS_OK && token != nullptr) rc = launch_append(*token, BF ? TS_BF16 : TS_F16, E4M3 ? TS_CACHE_E4M3 : TS_CACHE_INT8, 1, st);
  if (rc != TS_OK) return rc;
  TS_CUDA_TRY(launch_after(k, sm_count() * C, kThreads, smem, st, token != nullptr, 0, km, vm, a));
  TS_LAUNCH_CHECK();
  return TS_OK;
}

template <bool BF, bool E4M3>
static int launch(const AttnArgs& a, const AppendArgs* token, cudaStream_t st) {
  // one column tile of eight query heads, or two where a group has more
  const bool wide = a.group > 8;
  if (a.c.head_dim <= 64) return wide ? launch<BF, E4M3, 64, 2, 3>(a, token, st) : launch<BF, E4M3, 64, 1, 4>(a, token, st);
  if (a.c.head_dim <= 96) return wide ? launch<BF, E4M3, 96, 2, 2>(a, token, st) : launch<BF, E4M3, 96, 1, 3>(a, token, st);
  if (a.c.head_dim <= 128) {
    if (wide) return launch<BF, E4M3, 128, 2, 2>(a, token, st);
    const bool many = (int64_t)a.c.batch * a.c.n_kv >= (int64_t)kManyRows * sm_count() &&
                      (int64_t)a.c.max_pages * a.c.page_size <= kShortTable;
    return many ? launch<BF, E4M3, 128, 1, 3>(a, token, st) : launch<BF, E4M3, 128, 1, 2>(a, token, st);
  }
  return wide ? launch<BF, E4M3, 256, 2, 1>(a, token, st) : launch<BF, E4M3, 256, 1, 1>(a, token, st);
}

// Fills `a` from the arguments that both entry points share, and checks them.
static int make_args(AttnArgs* a, int q_dtype, int n_q, const ts_paged_cache8* cache, const int64_t* positions,
                     const float* rope_cos, const float* rope_sin, int64_t rope_rows, float scale, void* out,
                     int64_t out_row_stride, void* workspace, size_t workspace_bytes) {
  const int rc = make_cache(cache, &a->c);
  if (rc != TS_OK) return rc;
  TS_UNSUPPORTED(q_dtype == TS_F16 || q_dtype == TS_BF16, "queries must be fp16 or bf16");
  TS_REQUIRE((rope_cos == nullptr) == (rope_sin == nullptr), "rope_cos and rope_sin come both or neither");
  TS_REQUIRE(n_q > 0 && n_q % a->c.n_kv == 0, "bad head counts");
  TS_REQUIRE(scale > 0.f && scale < INFINITY, "scale must be positive and finite");
  TS_REQUIRE(is_aligned(out, 4) && out_row_stride % 2 == 0, "rows of out must be 4-byte aligned");
  if (a->c.batch == 0) return TS_OK;
  TS_REQUIRE(out, "NULL pointer");
  TS_REQUIRE(positions != nullptr || rope_cos == nullptr, "positions are needed for the rotation");
  a->group = n_q / a->c.n_kv;
  const int heads = a->group > 8 ? 16 : 8;
  a->head_tiles = (a->group + heads - 1) / heads;
  // Where a token's heads lie next to each other, up to four CTAs of neighbouring numbers
  // take as many heads of the same slots at about the same time, so that DRAM serves longer
  // runs: 64 sequences of up to 8191 slots 102 us for 112 (two heads 103, eight 102). Pages of
  // whole heads gain nothing (57 us for 57) and keep all CTAs.
  a->abreast = 1;
  for (int n = 2; n <= 4; ++n)
    if (a->c.head_stride < a->c.token_stride && a->c.n_kv * a->head_tiles % n == 0) a->abreast = n;
  TS_UNSUPPORTED((int64_t)a->c.batch * a->c.n_kv * a->head_tiles < (int64_t)kCounters, "too many heads in one call");
  TS_UNSUPPORTED(((int64_t)a->c.max_pages * a->c.page_size / kUnit + 1 + kRowCost) * a->c.batch * a->c.n_kv * a->head_tiles <
                     (int64_t)1 << 31,
                 "too many slots in one call");
  if (workspace == nullptr || workspace_bytes < workspace_bytes_of(a->c.head_dim)) {
    set_error("workspace of %zu bytes, %zu needed", workspace_bytes, workspace_bytes_of(a->c.head_dim));
    return TS_ERR_WORKSPACE;
  }
  TS_REQUIRE(is_aligned(workspace, 16), "workspace must be 16-byte aligned");
  a->n_q = n_q;
  a->positions = positions;
  a->cos_t = rope_cos;
  a->sin_t = rope_sin;
  a->rope_rows = rope_rows;
  a->scale2 = scale * 1.4426950408889634f;
  a->out = reinterpret_cast<uint16_t*>(out);
  a->out_stride = out_row_stride;
  a->counters = reinterpret_cast<int*>(workspace);
  a->partials = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + kCounterBytes);
  a->page_shift = log2_of(a->c.page_size);
  a->whole_pairs = a->c.page_size % kPair == 0 ? 1 : 0;
  a->wait_ns = wait_limit_ns();
  a->stall = take_test_stall() ? 1 : 0;
  return TS_OK;
}

static int attend(const AttnArgs& a, const AppendArgs* token, int dtype, int code, cudaStream_t st) {
  if (dtype == TS_BF16) return code == TS_CACHE_E4M3 ? launch<true, true>(a, token, st) : launch<true, false>(a, token, st);
  return code == TS_CACHE_E4M3 ? launch<false, true>(a, token, st) : launch<false, false>(a, token, st);
}

}  // namespace paged8
}  // namespace ts

using namespace ts;

extern "C" size_t ts_paged8_attention_workspace_size(const ts_paged_cache8* cache, int n_q) {
  (void)n_q;
  return cache == nullptr ? 0 : paged8::workspace_bytes_of(cache->head_dim);
}

extern "C" int ts_paged8_attention(const void* q, int q_dtype, int64_t q_row_stride, int n_q, const ts_paged_cache8* cache,
                                   const int64_t* positions, const float* rope_cos, const float* rope_sin,
                                   int64_t rope_rows, float scale, void* out, int64_t out_row_stride, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  paged8::AttnArgs a;
  const int rc = paged8::make_args(&a, q_dtype, n_q, cache, positions, rope_cos, rope_sin, rope_rows, scale, out, out_row_stride,
                                   workspace, workspace_bytes);
  if (rc != TS_OK || a.c.batch == 0) return rc;
  TS_REQUIRE(q && is_aligned(q, 2), "NULL or unaligned pointer");
  a.q = reinterpret_cast<const uint16_t*>(q);
  a.q_stride = q_row_stride;
  a.extra = 0;
  return paged8::attend(a, nullptr, q_dtype, cache->code, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int ts_paged8_decode_attention(const void* qkv, int qkv_dtype, int64_t qkv_row_stride, int n_q,
                                          const ts_paged_cache8* cache, const int64_t* positions, const float* rope_cos,
                                          const float* rope_sin, int64_t rope_rows, float scale, void* out,
                                          int64_t out_row_stride, void* workspace, size_t workspace_bytes, void* stream) {
  paged8::AttnArgs a;
  const int rc = paged8::make_args(&a, qkv_dtype, n_q, cache, positions, rope_cos, rope_sin, rope_rows, scale, out, out_row_stride,
                             workspace, workspace_bytes);
  if (rc != TS_OK || a.c.batch == 0) return rc;
  TS_REQUIRE(qkv && is_aligned(qkv, 16) && qkv_row_stride % 8 == 0, "qkv rows must be 16-byte aligned");
  a.q = reinterpret_cast<const uint16_t*>(qkv);
  a.q_stride = qkv_row_stride;
  a.extra = 1;
  paged8::AppendArgs p;
  p.c = a.c;
  p.k = a.q + (int64_t)n_q * a.c.head_dim;
  p.v = p.k + (int64_t)a.c.n_kv * a.c.head_dim;
  p.kb = p.vb = qkv_row_stride;
  p.kt = p.vt = 0;
  p.kh = p.vh = a.c.head_dim;
  p.tokens = 1;
  p.offsets = nullptr;
  p.n_new = nullptr;
  p.first = positions;
  p.cos_t = rope_cos;
  p.sin_t = rope_sin;
  p.rope_rows = rope_rows;
  return paged8::attend(a, &p, qkv_dtype, cache->code, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int ts_paged8_status(int clear, void* stream) {
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int v = 0;
  TS_CUDA_TRY(cudaMemcpyFromSymbolAsync(&v, paged8::g_err, sizeof(int), 0, cudaMemcpyDeviceToHost, st));
  TS_CUDA_TRY(cudaStreamSynchronize(st));
  if (v == 0) return TS_OK;
  if (clear) {
    const int zero = 0;
    TS_CUDA_TRY(cudaMemcpyToSymbolAsync(paged8::g_err, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st));
    TS_CUDA_TRY(cudaStreamSynchronize(st));
  }
  set_error("a bounded wait in the 8-bit attention ran out (code %d); the outputs of the calls since the last "
            "status check are not valid", v);
  return TS_ERR_TIMEOUT;
}
