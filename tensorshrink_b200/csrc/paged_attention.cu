// Attention of one new token per sequence over a paged key-value cache.
//
//   q, k, v of the new token from its projection; q and k rotated to the
//   token's position; k and v stored in slot len of the sequence; then, for
//   each query head of the kv head's group,
//     s_t = scale q . k_t,  t = 0 .. len,      p = softmax(s),   o = sum_t p_t v_t
//   and, when weights are accumulated, score_t += sum over the group of p_t
//   (the new slot's score is set, not added to).
//
// What bounds it: the cache is read once, 2 len D elements per kv head, and
// every element meets only the group's few query heads, so DRAM bandwidth
// does. The work is cut into units of 64 slots of one kv head, the units of
// all sequences laid end to end, and CTA i takes an equal range of them: a
// batch of unequal lengths, or a single long sequence, loads every SM alike.
// A head whose units lie in several CTAs is joined by the last of them to
// arrive, from fp32 partial sums in the workspace, in CTA order (so results
// do not depend on timing).
//
// Inside a CTA each warp owns 16 slots of every unit and streams them through
// its own ring of shared-memory stages with cp.async (no CTA barrier in the
// loop). Scores and outputs use mma.m16n8k16 with the group's heads as the 16
// rows: padding a small group to 16 rows costs tensor-core time that the
// kernel has to spare, and P passes from the score accumulators to the second
// product without leaving registers. Softmax statistics and sums are fp32. P
// enters its product as two terms of the cache's type (16 bits of it): one
// alone would add as large an error as the rounding of the output does, and
// the second product costs nothing that the loads do not hide. (Making every v
// of the second product finite instead of its weights positive cost 6%.)
//
// Measured (bf16, 128 columns, 8 kv heads of 4 query heads): 64 sequences of up to
// 8191 slots, 177 us, 6.1 TB/s, 94% of the copy bandwidth; 4 of 32768, 88 us, with
// the logits kept 90 to 92 us (98 us with the cache read at the same L2 priority as
// the logits are written); one of 512, 10.0 us, a chain of latencies (lengths,
// pages, rows, the warps' and the CTAs' joins).
#include <algorithm>

#include "paged_split.cuh"

namespace ts {
namespace paged {

constexpr int kHeads = 16;                 // query heads of an MMA tile

struct AttnArgs {
  Cache c;
  const uint16_t* qkv;
  int64_t qkv_stride;
  int n_q, group, head_tiles;
  const int64_t* positions;
  const float* cos_t;
  const float* sin_t;
  int64_t rope_rows;
  float scale2;          // scale * log2(e)
  uint16_t* out;
  int64_t out_stride;
  int* counters;
  float* partials;       // [grid][2][16][D + 2]: the group's rows, each with its max and sum
  float* lse2;           // [batch * n_q] log2 of the softmax denominators, or NULL
  float* logits;         // [batch * n_q][cap] scores in log2 units, or NULL
  int64_t logit_stride;
  int page_shift;        // log2(page_size), or -1
  int one_page;          // page_size % 16 == 0: a warp's 16 slots share a page
};

// s / page_size and s % page_size.
__device__ __forceinline__ void split_slot(const AttnArgs& a, int s, int* page, int* off) {
  if (a.page_shift >= 0) {
    *page = s >> a.page_shift;
    *off = s & (a.c.page_size - 1);
  } else {
    *page = s / a.c.page_size;
    *off = s - *page * a.c.page_size;
  }
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Units of a sequence of `len` cached tokens for one kv head; 0 without a
// slot for the new one.
__device__ __forceinline__ int units_of(const AttnArgs& a, int len) {
  return len < 0 || len >= capacity(a.c) ? 0 : len / kUnit + 1;
}

// Whether sequence b, with a slot for its new token, can take it: the slot
// has memory and the position a row in the rotary tables.
__device__ __forceinline__ bool takes(const AttnArgs& a, int b, int len, int64_t pos) {
  int pg, off;
  split_slot(a, len, &pg, &off);
  const int page = a.c.table[b * a.c.table_stride + pg];
  return (unsigned)page < (unsigned)a.c.num_pages && (a.cos_t == nullptr || (pos >= 0 && pos < a.rope_rows));
}

// A pair of weights rounded towards zero, and a pair made at least the type's
// smallest number (bf16: 2^-133, fp16: 2^-24).
template <bool BF>
__device__ __forceinline__ uint32_t pack2_down(float a, float b) {
  uint32_t d;
  if (BF) asm("cvt.rz.bf16x2.f32 %0, %2, %1;" : "=r"(d) : "f"(a), "f"(b));
  else asm("cvt.rz.f16x2.f32 %0, %2, %1;" : "=r"(d) : "f"(a), "f"(b));
  return d;
}
template <bool BF>
__device__ __forceinline__ uint32_t positive2(uint32_t w) {
  if (BF) asm("max.bf16x2 %0, %0, %1;" : "+r"(w) : "r"(0x00010001u));
  else asm("max.f16x2 %0, %0, %1;" : "+r"(w) : "r"(0x00010001u));
  return w;
}

// Shared memory: the warps' rings [kWarps][S][K, V][16 rows][pitch], the
// query tile [16][DP + 8] and the prefix sums of the sequences' units. Row r
// keeps its 16-byte chunk c at c ^ (r & 7), so that ldmatrix reads of eight
// rows touch every bank once.
template <int DP>
constexpr int stages_for() { return DP == 64 ? 4 : 3; }
template <int DP>
constexpr size_t ring_bytes() { return (size_t)kWarps * stages_for<DP>() * 2 * kRows * DP * 2; }
template <int DP>
constexpr size_t attn_smem(int batch) {
  return ring_bytes<DP>() + kHeads * (DP + 8) * 2 + (size_t)(2 * batch + 1) * 4;
}

template <bool BF, int DP>
__global__ void __launch_bounds__(kThreads, DP == 64 ? 3 : DP == 128 ? 2 : 1) paged_attention_kernel(const AttnArgs a) {
  constexpr int S = stages_for<DP>();
  constexpr int kPitch = DP * 2;                 // bytes of a staged row
  constexpr int kStage = 2 * kRows * kPitch;     // bytes of a stage: K rows, then V rows
  constexpr int kSteps = DP / 16;
  constexpr bool kKeepQ = DP <= 128;             // query fragments stay in registers
  constexpr float kShift = BF ? 0.f : 15.f;      // weights and their sums are 2^kShift times: fp16 holds them down to 2^-39
  constexpr int kRowChunks = DP / 8;             // 16-byte columns of a staged row
  constexpr int kRowsPer = 32 / kRowChunks;      // rows that a warp copies at once
  extern __shared__ __align__(1024) char smem[];
  uint16_t* qs = reinterpret_cast<uint16_t*>(smem + ring_bytes<DP>());
  int* prefix = reinterpret_cast<int*>(smem + ring_bytes<DP>() + kHeads * (DP + 8) * 2);   // [batch + 1]
  __shared__ uint64_t warp_sums[kWarps];
  __shared__ int warp_most[kWarps];
  __shared__ int is_last;
  pdl_launch_dependents();                             // the weights' kernel may take its place in the queue
  const Cache& c = a.c;
  int* lens = prefix + c.batch + 1;                                                        // [batch]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int D = c.head_dim, chunks = D / 8, steps = D / 16, rows_per_b = c.n_kv * a.head_tiles;

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
    // How the units are dealt out (`deal`): a row of n units counts n + front,
    // or, with front < 0, -front whatever n is.
    const unsigned units = (unsigned)(uint32_t)all * rows_per_b, rows = (unsigned)(all >> 32) * rows_per_b;
    deal = choose_deal(units, rows, longest, gridDim.x, min(a.group, kHeads));
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
  // rows of the query tile that no head fills: zeros, so that their scores are finite
  for (int i = tid; i < kHeads * (DP + 8) / 2; i += kThreads) reinterpret_cast<uint32_t*>(qs)[i] = 0;
  __syncthreads();
  // a sequence that the call cannot take answers with zeros
  for (int b = blockIdx.x; b < c.batch; b += gridDim.x)
    if (prefix[b] == prefix[b + 1])
      for (int i = tid; i < a.n_q * D; i += kThreads) a.out[b * a.out_stride + i] = 0;

  const unsigned total = (unsigned)prefix[c.batch] * rows_per_b;   // (the host keeps it below 2^31)
  if (total == 0) return;
  const unsigned n_cta = min(deal.n_cta, total);
  if (blockIdx.x >= n_cta) return;
  const Shares shares(total, n_cta);
  const unsigned u1 = shares.begin(blockIdx.x + 1);

  // with scores to accumulate, the logits shall stay in L2, not the cache
  uint64_t policy;
  if (a.logits != nullptr) asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
  else asm("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
  char* ring = smem + (size_t)warp * S * kStage;
  const uint32_t ring_u = smem_u32(ring);
  const uint32_t qs_u = smem_u32(qs);

  // the first row: sequence b is the last with prefix[b] * rows_per_b <= u
  unsigned u = shares.begin(blockIdx.x);
  int b = 0;
  for (int hi = c.batch - 1; b < hi;) {
    const int mid = (b + hi + 1) >> 1;
    if ((unsigned)prefix[mid] * rows_per_b <= u) b = mid; else hi = mid - 1;
  }
  int row = (int)((u - (unsigned)prefix[b] * rows_per_b) / (unsigned)(prefix[b + 1] - prefix[b]));
  for (; u < u1; ++row) {
    // the segment: units [t0, t1) of (sequence b, kv head h, head tile ht)
    if (row == rows_per_b) {
      row = 0;
      do ++b; while (prefix[b + 1] == prefix[b]);
    }
    const int cost = prefix[b + 1] - prefix[b], nt = units_of(a, lens[b]), front = cost - nt;
    const unsigned row_u = (unsigned)prefix[b] * rows_per_b + (unsigned)(row * cost);
    const int v0 = (int)(u - row_u), v1 = (int)min((unsigned)cost, v0 + (u1 - u));
    u += v1 - v0;
    if (v1 <= front) continue;                         // only the row's front
    const int t0 = max(v0 - front, 0), t1 = v1 - front;
    const int h = row / a.head_tiles, ht = row - h * a.head_tiles;
    const int heads = min(kHeads, a.group - ht * kHeads);
    const int head0 = h * a.group + ht * kHeads;       // first query head of the tile
    const int len = lens[b];
    const int32_t* table = c.table + b * c.table_stride;
    const uint16_t* new_row = a.qkv + b * a.qkv_stride;
    const bool turn = a.cos_t != nullptr;

    // What the segment needs first is loaded before any of it is used: the
    // position, the new token's page, the first stages' pages, the query heads
    // (kQ of a thread at a time; behind the copies they would wait).
    constexpr int kQ = 4;
    const int64_t pos_in = a.positions != nullptr ? a.positions[b] : 0;
    int pg_new, off_new;
    split_slot(a, len, &pg_new, &off_new);
    const int page_new = table[pg_new];
    auto page_at = [&](int t) {                        // (one_page) the page of unit t's rows
      const int slot0 = t * kUnit + warp * kRows;
      int pg, off;
      split_slot(a, slot0, &pg, &off);
      return t < t1 && slot0 < len ? table[pg] : -1;
    };
    int pages[S];
#pragma unroll
    for (int s = 0; s < S; ++s) pages[s] = a.one_page ? page_at(t0 + s) : -1;
    const int qj = tid % (DP / 2), q_first = tid / (DP / 2);   // this thread's column pair and first head
    constexpr int kQStep = kThreads / (DP / 2);                 // heads that the threads cover at once
    uint32_t qx[kQ];
    auto load_q = [&](int g0) {
#pragma unroll
      for (int k = 0; k < kQ; ++k) {
        const int g = g0 + k * kQStep;
        if (qj < D / 2 && g < heads) {
          const uint16_t* qr = new_row + (int64_t)(head0 + g) * D + qj;
          qx[k] = (uint32_t)qr[0] | ((uint32_t)qr[D / 2] << 16);
        }
      }
    };
    load_q(q_first);
    // a sequence that cannot take its token answers with zeros
    const bool ok = (unsigned)page_new < (unsigned)c.num_pages && (!turn || (pos_in >= 0 && pos_in < a.rope_rows));
    const int64_t pos = ok ? pos_in : 0;
    const float* cs = a.cos_t + pos * (D / 2);
    const float* sn = a.sin_t + pos * (D / 2);
    float2 rot = make_float2(1.f, 0.f);
    if (turn && qj < D / 2) rot = make_float2(cs[qj], sn[qj]);

    // A warp's share of unit t: slots t * 64 + warp * 16 + r. It copies the
    // rows of cached slots and zeros for the others; `live` is a bit per row
    // that has a cached token, queued until the stage is consumed.
    const int cl = lane % kRowChunks, rl = lane / kRowChunks;   // this lane's 16-byte column and first row
    const bool col = cl < chunks;
    auto issue = [&](int t, int stage, int page) -> uint32_t {
      uint32_t live = 0;
      if (t < t1) {
        const int slot0 = t * kUnit + warp * kRows;
        const uint32_t dst = ring_u + stage * kStage + rl * kPitch;
        const int n = min(kRows, len - slot0);          // rows with cached tokens
        if (a.one_page) {
          int pg, off;
          split_slot(a, slot0, &pg, &off);
          const int rows = (unsigned)page < (unsigned)c.num_pages ? n : 0;
          live = rows > 0 ? (1u << rows) - 1 : 0;
          // row 2 i + rl of a 256-byte row (and alike for the other widths):
          // its swizzled column is this lane's with bits of i flipped
          const uint32_t x0 = (uint32_t)(cl ^ rl) << 4;
          const int64_t e = rows > 0 ? (row_at(c, page, h, off + rl) + cl * 8) * 2 : 0;
          const char* kp = c.k + e;
          const int64_t step = c.token_stride * (kRowsPer * 2), kv = c.v - c.k;
          if (rows == kRows) {
            if (col) {
#pragma unroll
              for (int i = 0; i < kRows / kRowsPer; ++i) {
                const uint32_t d = dst + i * kRowsPer * kPitch + (x0 ^ (((i * kRowsPer) & 7) << 4));
                cp16(d, kp, policy);
                cp16(d + kRows * kPitch, kp + kv, policy);
                kp += step;
              }
            }
          } else if (col) {
#pragma unroll
            for (int i = 0; i < kRows / kRowsPer; ++i) {
              const int ok = i * kRowsPer + rl < rows;
              const uint32_t d = dst + i * kRowsPer * kPitch + (x0 ^ (((i * kRowsPer) & 7) << 4));
              cp16(d, ok ? kp : c.k, ok * 16, policy);
              cp16(d + kRows * kPitch, ok ? kp + kv : c.v, ok * 16, policy);
              if (ok) kp += step;
            }
          }
        } else {
          // pages may end inside the rows: lane r (< 16) looks row r up
          const int r0 = lane & 15;
          int64_t o = -1;
          if (r0 < n) {
            int pg, off;
            split_slot(a, slot0 + r0, &pg, &off);
            const int p = table[pg];
            if ((unsigned)p < (unsigned)c.num_pages) o = row_at(c, p, h, off);
          }
          live = __ballot_sync(0xffffffffu, o >= 0) & 0xFFFFu;
#pragma unroll
          for (int i = 0; i < kRows / kRowsPer; ++i) {
            const int r = i * kRowsPer + rl;
            const int64_t ro = __shfl_sync(0xffffffffu, o, r);
            const int ok = ro >= 0;
            const int64_t e = ok ? (ro + cl * 8) * 2 : 0;
            const uint32_t d = dst + i * kRowsPer * kPitch + ((cl ^ (r & 7)) << 4);
            if (col) {
              cp16(d, c.k + e, ok * 16, policy);
              cp16(d + kRows * kPitch, c.v + e, ok * 16, policy);
            }
          }
        }
      }
      cp_commit();
      return live;
    };
    uint64_t live_q = 0;
#pragma unroll
    for (int s = 0; s < S - 1; ++s) live_q |= (uint64_t)issue(t0 + s, s, pages[s]) << (16 * s);
    int page_next = pages[S - 1];

    // the rotated query heads of the tile
    for (int g0 = q_first; g0 < heads; g0 += kQ * kQStep) {
      if (g0 != q_first) load_q(g0);
#pragma unroll
      for (int k = 0; k < kQ; ++k) {
        const int g = g0 + k * kQStep;
        if (qj >= D / 2 || g >= heads) continue;
        if (turn) {
          const float2 f = unpack2<BF>(qx[k]);
          const float2 y = rotate(f.x, f.y, rot.x, rot.y);
          qx[k] = pack2<BF>(y.x, y.y);
        }
        qs[g * (DP + 8) + qj] = (uint16_t)qx[k];
        qs[g * (DP + 8) + qj + D / 2] = (uint16_t)(qx[k] >> 16);
      }
    }
    __syncthreads();
    uint32_t qf[kKeepQ ? kSteps : 1][4];
    const uint32_t q_addr = qs_u + ((lane & 15) * (DP + 8) + (lane >> 4) * 8) * 2;
    if (kKeepQ) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        if (s < steps) ldsm4(q_addr + s * 32, qf[kKeepQ ? s : 0]);
    }

    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const int r7 = lane & 7;

    int stage = 0;
    for (int t = t0; t < t1; ++t) {
      live_q |= (uint64_t)issue(t + S - 1, stage == 0 ? S - 1 : stage - 1, page_next) << (16 * (S - 1));
      if (a.one_page) page_next = page_at(t + S);
      uint32_t live = (uint32_t)live_q & 0xFFFFu;
      live_q >>= 16;
      cp_wait<S - 1>();
      __syncwarp();
      const int slot0 = t * kUnit + warp * kRows;
      const uint32_t kb = ring_u + stage * kStage, vb = kb + kRows * kPitch;
      stage = stage + 1 == S ? 0 : stage + 1;
      if (slot0 > len) continue;                       // warp-uniform: nothing left for this warp
      if (ok && len < slot0 + kRows) {
        // the new token's row: into the stage and, once per kv head, the cache
        const int r = len - slot0;
        live |= 1u << r;
        char* st = ring + (kb - ring_u);
        const int64_t at = row_at(c, page_new, h, off_new);
        uint16_t* kc = reinterpret_cast<uint16_t*>(c.k) + at;
        uint16_t* vc = reinterpret_cast<uint16_t*>(c.v) + at;
        const uint16_t* kr = new_row + (int64_t)(a.n_q + h) * D;
        const uint16_t* vr = new_row + (int64_t)(a.n_q + c.n_kv + h) * D;
        for (int j = lane; j < D / 2; j += 32) {
          uint16_t x1 = kr[j], x2 = kr[j + D / 2];
          if (turn) {
            const float2 f = unpack2<BF>((uint32_t)x1 | ((uint32_t)x2 << 16));
            const float2 y = rotate(f.x, f.y, cs[j], sn[j]);
            const uint32_t p = pack2<BF>(y.x, y.y);
            x1 = (uint16_t)p;
            x2 = (uint16_t)(p >> 16);
          }
          const uint16_t v1 = vr[j], v2 = vr[j + D / 2];
          const int j2 = j + D / 2;
          auto at16 = [&](int e) { return r * kPitch + (((e >> 3) ^ (r & 7)) << 4) + (e & 7) * 2; };
          *reinterpret_cast<uint16_t*>(st + at16(j)) = x1;
          *reinterpret_cast<uint16_t*>(st + at16(j2)) = x2;
          *reinterpret_cast<uint16_t*>(st + kRows * kPitch + at16(j)) = v1;
          *reinterpret_cast<uint16_t*>(st + kRows * kPitch + at16(j2)) = v2;
          if (ht == 0) {
            kc[j] = x1;
            kc[j2] = x2;
            vc[j] = v1;
            vc[j2] = v2;
          }
        }
        if (lane == 0 && ht == 0) {
          const int64_t sa = stat_at(c, page_new, h, off_new);
          if (c.scores != nullptr) c.scores[sa] = 0.f;
          if (c.slot_pos != nullptr) c.slot_pos[sa] = (int32_t)pos;
        }
        __syncwarp();
      }

      // scores of 16 heads x 16 slots
      float sc[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
      const int krow = (lane & 7) + ((lane >> 4) << 3);
      const uint32_t k_addr = (kb + krow * kPitch) | ((((lane >> 3) & 1) ^ r7) << 4);   // rows start at multiples of their pitch
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (s >= steps) break;
        uint32_t kf[4];
        ldsm4(k_addr ^ (s << 5), kf);
        if (!kKeepQ) ldsm4(q_addr + s * 32, qf[0]);
        mma<BF>(sc[0], qf[kKeepQ ? s : 0], kf[0], kf[1]);
        mma<BF>(sc[1], qf[kKeepQ ? s : 0], kf[2], kf[3]);
      }
      const int c0 = (lane & 3) * 2;
      if (live != 0xFFFFu) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!((live >> (n * 8 + c0 + (e & 1))) & 1)) sc[n][e] = -INFINITY;
      }
      if (a.logits != nullptr) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int g = (lane >> 2) + 8 * e;
          if (g < heads) {
            float* lg = a.logits + (int64_t)(b * a.n_q + head0 + g) * a.logit_stride + slot0 + c0;
            *reinterpret_cast<float2*>(lg) = make_float2(sc[0][2 * e] * a.scale2, sc[0][2 * e + 1] * a.scale2);
            *reinterpret_cast<float2*>(lg + 8) = make_float2(sc[1][2 * e] * a.scale2, sc[1][2 * e + 1] * a.scale2);
          }
        }
      }
      // online softmax of the two rows this thread holds parts of; m and the
      // maxima are unscaled, weights are 2^(s scale2 - m scale2)
      float mn[2], base[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = fmaxf(fmaxf(sc[0][2 * e], sc[0][2 * e + 1]), fmaxf(sc[1][2 * e], sc[1][2 * e + 1]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        mn[e] = fmaxf(m[e], x);
        base[e] = mn[e] == -INFINITY ? 0.f : mn[e] * a.scale2;
      }
      if (__any_sync(0xffffffffu, mn[0] > m[0] || mn[1] > m[1])) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float corr = ex2(fmaf(m[e], a.scale2, -base[e]));
          l[e] *= corr;
#pragma unroll
          for (int i = 0; i < DP / 8; ++i) {
            o[i][2 * e] *= corr;
            o[i][2 * e + 1] *= corr;
          }
          m[e] = mn[e];
        }
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[n][e] = ex2(fmaf(sc[n][e], a.scale2, kShift - base[e >> 1]));
      l[0] += (sc[0][0] + sc[0][1]) + (sc[1][0] + sc[1][1]);
      l[1] += (sc[0][2] + sc[0][3]) + (sc[1][2] + sc[1][3]);
      // P in two terms of the cache's type, the first rounded towards zero and the
      // second positive, so that an infinite v comes out of both as itself (a
      // second term of 0, or of the other sign, would make it NaN)
      uint32_t pf[4], pr[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = sc[i >> 1][2 * (i & 1)], y = sc[i >> 1][2 * (i & 1) + 1];
        pf[i] = pack2_down<BF>(x, y);
        const float2 h = unpack2<BF>(pf[i]);
        pr[i] = positive2<BF>(pack2<BF>(x - h.x, y - h.y));
      }
      const int vrow = lane & 15;
      const uint32_t v_addr = (vb + vrow * kPitch) | (((lane >> 4) ^ r7) << 4);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (s >= steps) break;
        uint32_t vf[4];
        ldsm4t(v_addr ^ (s << 5), vf);
        mma<BF>(o[2 * s], pf, vf[0], vf[1]);
        mma<BF>(o[2 * s + 1], pf, vf[2], vf[3]);
        mma<BF>(o[2 * s], pr, vf[0], vf[1]);
        mma<BF>(o[2 * s + 1], pr, vf[2], vf[3]);
      }
      __syncwarp();   // the stage is refilled at the top of the next round
    }
    cp_wait<0>();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }
    __syncthreads();

    // join the warps through shared memory (over the drained rings)
    constexpr int kJoin = DP + 4;                    // floats of a row: its sums, max, sum
    float* jo = reinterpret_cast<float*>(smem);      // [kWarps][16][kJoin]
    static_assert((size_t)kWarps * kHeads * (kJoin + 2) * 4 <= ring_bytes<DP>(), "join area");
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float* r = jo + (warp * kHeads + (lane >> 2) + 8 * e) * kJoin;
#pragma unroll
      for (int i = 0; i < DP / 8; ++i)
        *reinterpret_cast<float2*>(r + i * 8 + (lane & 3) * 2) = make_float2(o[i][2 * e], o[i][2 * e + 1]);
      if ((lane & 3) == 0) {
        r[DP] = m[e] * a.scale2;                       // in log2 units from here on
        r[DP + 1] = l[e];
      }
    }
    __syncthreads();
    // factors 2^(m_warp - m) of every warp and head, then the sums
    float* fac = jo + kWarps * kHeads * kJoin;       // [kWarps][16], then [16] maxima, [16] sums
    if (tid < kHeads) {
      float wm[kWarps], mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, wm[w] = jo[(w * kHeads + tid) * kJoin + DP]);
      const float bs = mm == -INFINITY ? 0.f : mm;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(wm[w] - bs);
        fac[w * kHeads + tid] = f;
        ll = fmaf(f, jo[(w * kHeads + tid) * kJoin + DP + 1], ll);
      }
      fac[kWarps * kHeads + tid] = mm;
      fac[(kWarps + 1) * kHeads + tid] = ll;
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == nt;
    const int64_t prow = (int64_t)kHeads * (D + 2);  // a piece: [16][D] sums, [16] (max, sum)
    // a CTA has at most two partial rows: one that it ends, one that it begins
    float* part = a.partials + ((int64_t)blockIdx.x * 2 + (t0 > 0 ? 0 : 1)) * prow;
    uint16_t* out = a.out + b * a.out_stride + (int64_t)head0 * D;
    for (int i = tid; i < heads * (D / 4); i += kThreads) {
      const int g = i / (D / 4), d = 4 * (i - g * (D / 4));
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(jo + (w * kHeads + g) * kJoin + d);
        const float f = fac[w * kHeads + g];
        acc.x = fmaf(f, v.x, acc.x);
        acc.y = fmaf(f, v.y, acc.y);
        acc.z = fmaf(f, v.z, acc.z);
        acc.w = fmaf(f, v.w, acc.w);
      }
      if (whole) {
        const float inv = 1.f / fac[(kWarps + 1) * kHeads + g];
        uint32_t* dst = reinterpret_cast<uint32_t*>(out + g * D + d);
        dst[0] = ok ? pack2<BF>(acc.x * inv, acc.y * inv) : 0;
        dst[1] = ok ? pack2<BF>(acc.z * inv, acc.w * inv) : 0;
      } else {
        *reinterpret_cast<float4*>(part + g * D + d) = acc;
      }
    }
    if (tid < heads) {
      const float mm = fac[kWarps * kHeads + tid], ll = fac[(kWarps + 1) * kHeads + tid];
      if (!whole) reinterpret_cast<float2*>(part + kHeads * D)[tid] = make_float2(mm, ll);
      else if (a.lse2 != nullptr) a.lse2[b * a.n_q + head0 + tid] = mm + (log2f(ll) - kShift);
    }
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
        const float* begun = a.partials + ((int64_t)cta0 * 2 + 1) * prow;
        const float* others = a.partials + (int64_t)cta0 * 2 * prow;
        auto piece = [&](int i) { return i == 0 ? begun : others + (int64_t)i * 2 * prow; };
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
          float f[2][kML], inv[2];
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
                f[e][k] = ex2(ml[e][k].x - bs);
                ll = fmaf(f[e][k], ml[e][k].y, ll);
              }
              ll = warp_sum(ll);
              inv[e] = 1.f / ll;
              if (lane == 0 && a.lse2 != nullptr && g0 + e * kWarps < heads)
                a.lse2[b * a.n_q + head0 + g0 + e * kWarps] = bs + (log2f(ll) - kShift);
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
                  float w = f[e][0];
#pragma unroll
                  for (int k = 1; k < kML; ++k) w = i0 >= 32 * k ? f[e][k] : w;
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
    __syncthreads();   // the join area becomes the rings again
  }
}

// score[slot] += sum over the group of 2^(logit - lse2): a thread takes W
// neighbouring slots of a kv head, W = 4 where pages hold a multiple of four.
// Reads 4 bytes per slot and query head, next to the 4 D bytes per slot that
// the attention read, from L2: 8 us behind the attention of 4 x 32768 slots of 8
// kv heads of 4.
template <int W>
__global__ void __launch_bounds__(256, 6) paged_weights_kernel(const AttnArgs a) {
  const Cache& c = a.c;
  const int row = blockIdx.y, b = row / c.n_kv, h = row - b * c.n_kv;
  const int len = c.seq_lens[b];
  if (units_of(a, len) == 0) {
    // Every thread waits for the attention before it ends, those without a
    // slot too: where no sequence takes part nobody else would, and whatever
    // follows this kernel would not find the attention's zeros in `out`.
    pdl_wait_primary();
    return;
  }
  const bool ok = takes(a, b, len, a.positions != nullptr ? a.positions[b] : 0);
  const int64_t q = (int64_t)b * a.n_q + h * a.group;
  bool waits = true;
  for (int slot0 = (blockIdx.x * blockDim.x + threadIdx.x) * W; slot0 <= len; slot0 += gridDim.x * blockDim.x * W) {
    // what the attention does not write is read while it may still run
    int pg, off;
    split_slot(a, slot0, &pg, &off);
    const int page = c.table[b * c.table_stride + pg];
    const bool has = ok && (unsigned)page < (unsigned)c.num_pages;
    float* s = c.scores + (has ? stat_at(c, page, h, off) : 0);
    float w[W];
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = has && slot0 + i < len ? s[i] : 0.f;
    if (waits) pdl_wait_primary();
    waits = false;
    const float* lg = a.logits + q * a.logit_stride + slot0;
    float sum[W];
#pragma unroll
    for (int i = 0; i < W; ++i) sum[i] = 0.f;
    for (int g0 = 0; g0 < a.group; g0 += 4) {
      float v[4][W], lse[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (g0 + g >= a.group) break;
        lse[g] = a.lse2[q + g0 + g];
        const float* src = lg + (g0 + g) * a.logit_stride;
        if (W == 4) {
          const float4 f = __ldcs(reinterpret_cast<const float4*>(src));
          v[g][0] = f.x; v[g][1 % W] = f.y; v[g][2 % W] = f.z; v[g][3 % W] = f.w;
        } else {
          v[g][0] = __ldcs(src);
        }
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (g0 + g >= a.group) break;
#pragma unroll
        for (int i = 0; i < W; ++i) sum[i] += ex2(v[g][i] - lse[g]);
      }
    }
    if (!has) continue;
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (slot0 + i <= len) s[i] = w[i] + sum[i];
  }
  if (waits) pdl_wait_primary();
}

// Stores tokens behind a sequence's cached ones: slot len + t of every kv
// head gets k (rotated when tables are given) and v; scores and positions
// are set. A warp takes four tokens of a head at a time, 16 bytes per lane
// and token. Bound by DRAM traffic: every row is read and written once. 16 x 4096
// tokens of 8 kv heads of 128 columns: 86 us, 6.2 TB/s; one token: 2.5 us.
constexpr int kTok = 4;

struct AppendArgs {
  Cache c;
  const uint16_t* k;
  const uint16_t* v;
  int64_t kb, kt, kh, vb, vt, vh;   // element strides of sequence, token, head
  const int64_t* first;
  const int32_t* n_new;
  int tokens;
  const float* cos_t;
  const float* sin_t;
  int64_t rope_rows;
  const float* scores;
  int64_t sb, sh, st;
  int page_shift;       // log2(page_size), or -1
};

template <bool BF, bool ROPE>
__global__ void __launch_bounds__(256, ROPE ? 2 : 4) paged_append_kernel(const AppendArgs a) {
  const Cache& c = a.c;
  const int lane = threadIdx.x & 31;
  const int D = c.head_dim, chunks = D / 8, half = chunks / 2;
  const int b = blockIdx.y, len = c.seq_lens[b];
  const int tokens = a.n_new != nullptr ? min(a.tokens, a.n_new[b]) : a.tokens;
  if (len < 0 || tokens <= 0) return;
  const int64_t first = a.first != nullptr ? a.first[b] : len;
  // neighbouring warps take neighbouring heads of the same kTok tokens: both
  // the tokens' rows and the pages are touched in runs
  const int items = (tokens + kTok - 1) / kTok * c.n_kv;
  for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < items; i += gridDim.x * 8) {
    const int h = i % c.n_kv, t0 = i / c.n_kv * kTok;
    int64_t at[kTok];
    const int ch0 = lane;
    for (int ch = ch0; ch < 2 * chunks || ch == ch0; ch += 32) {   // (every lane comes by once, for the look-up)
      const bool is_v = ch >= chunks;
      const int cc = is_v ? ch - chunks : ch;
      const bool hi = cc >= half;
      const bool turn = ROPE && !is_v;
      const uint16_t* src = is_v ? a.v + b * a.vb + h * a.vh : a.k + b * a.kb + h * a.kh;
      const int64_t step = is_v ? a.vt : a.kt;
      // the rows are on their way while the pages are looked up
      uint4 w[kTok], p[kTok];
#pragma unroll
      for (int i = 0; i < kTok; ++i)
        if (t0 + i < tokens && ch < 2 * chunks) {
          const uint16_t* r = src + (t0 + i) * step;
          w[i] = *reinterpret_cast<const uint4*>(r + cc * 8);
          if (turn) p[i] = *reinterpret_cast<const uint4*>(r + (hi ? cc - half : cc + half) * 8);
        }
      if (ch == ch0) {
        // lane i (< kTok) looks token i up
        const int t = t0 + lane;
        const int64_t slot = (int64_t)len + t, pos = first + t;
        int64_t mine = -1;
        if (lane < kTok && t < tokens && slot < capacity(c) && (!ROPE || (pos >= 0 && pos < a.rope_rows))) {
          const int pg = a.page_shift >= 0 ? (int)slot >> a.page_shift : (int)slot / c.page_size;
          const int page = c.table[b * c.table_stride + pg], off = (int)slot - pg * c.page_size;
          if ((unsigned)page < (unsigned)c.num_pages) {
            mine = row_at(c, page, h, off);
            const int64_t sa = stat_at(c, page, h, off);
            if (c.scores != nullptr) c.scores[sa] = a.scores != nullptr ? a.scores[b * a.sb + h * a.sh + t * a.st] : 0.f;
            if (c.slot_pos != nullptr) c.slot_pos[sa] = (int32_t)pos;
          }
        }
#pragma unroll
        for (int i = 0; i < kTok; ++i) at[i] = __shfl_sync(0xffffffffu, mine, i);
      }
      if (ch >= 2 * chunks) break;
#pragma unroll
      for (int i = 0; i < kTok; ++i) {
        if (at[i] < 0) continue;
        if (turn) {
          const int64_t j = (first + t0 + i) * (D / 2) + (hi ? cc - half : cc) * 8;
          const float* cs = a.cos_t + j;
          const float* sn = a.sin_t + j;
          uint32_t* ww = reinterpret_cast<uint32_t*>(&w[i]);
          const uint32_t* pw = reinterpret_cast<const uint32_t*>(&p[i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 x = unpack2<BF>(hi ? pw[e] : ww[e]), y = unpack2<BF>(hi ? ww[e] : pw[e]);
            const float2 r0 = rotate(x.x, y.x, cs[2 * e], sn[2 * e]);
            const float2 r1 = rotate(x.y, y.y, cs[2 * e + 1], sn[2 * e + 1]);
            ww[e] = hi ? pack2<BF>(r0.y, r1.y) : pack2<BF>(r0.x, r1.x);
          }
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(is_v ? c.v : c.k) + at[i] + cc * 8) = w[i];
      }
    }
  }
}

int make_cache(const ts_paged_cache* p, Cache* o) {
  TS_REQUIRE(p != nullptr, "NULL cache");
  // (of no sequences at all there may be no memory)
  TS_REQUIRE(p->batch == 0 || (p->k_pages && p->v_pages && p->page_table && p->seq_lens), "NULL pointer in the cache");
  TS_UNSUPPORTED(p->dtype == TS_F16 || p->dtype == TS_BF16, "the cache holds fp16 or bf16");
  TS_REQUIRE(p->batch >= 0 && p->n_kv > 0 && p->page_size > 0 && (p->batch == 0 || (p->num_pages > 0 && p->max_pages > 0)),
             "bad cache sizes");
  TS_UNSUPPORTED(p->head_dim % 16 == 0 && p->head_dim >= 16 && p->head_dim <= 256,
                 "head_dim must be a multiple of 16, <= 256");
  TS_REQUIRE((int64_t)p->max_pages * p->page_size <= (int64_t)1 << 30, "more than 2^30 slots per sequence");
  TS_REQUIRE(is_aligned(p->k_pages, 16) && is_aligned(p->v_pages, 16) && p->page_stride % 8 == 0 &&
                 p->head_stride % 8 == 0 && p->token_stride % 8 == 0,
             "cache rows must be 16-byte aligned");
  o->k = reinterpret_cast<char*>(p->k_pages);
  o->v = reinterpret_cast<char*>(p->v_pages);
  o->page_stride = p->page_stride;
  o->head_stride = p->head_stride;
  o->token_stride = p->token_stride;
  o->table = p->page_table;
  o->table_stride = p->table_stride;
  o->seq_lens = p->seq_lens;
  o->scores = p->scores;
  o->slot_pos = p->slot_pos;
  o->batch = p->batch;
  o->n_kv = p->n_kv;
  o->head_dim = p->head_dim;
  o->page_size = p->page_size;
  o->num_pages = p->num_pages;
  o->max_pages = p->max_pages;
  return TS_OK;
}

// log2 of a power of two, -1 of anything else.
int log2_of(int v) {
  for (int i = 0; i < 31; ++i)
    if (v == 1 << i) return i;
  return -1;
}

static size_t grid_of(int head_dim) { return (size_t)sm_count() * (head_dim > 128 ? 1 : head_dim > 64 ? 2 : 3); }

struct Layout {
  size_t partials, lse, logits, bytes;
  int64_t logit_stride;
};

static Layout attn_layout(const ts_paged_cache& p, int n_q, bool weights) {
  Layout L;
  L.partials = kCounterBytes;
  L.lse = align_up(L.partials + grid_of(p.head_dim) * 2 * kHeads * (p.head_dim + 2) * 4, 256);
  L.logits = align_up(L.lse + (weights ? (size_t)p.batch * n_q * 4 : 0), 256);
  L.logit_stride = (int64_t)align_up((size_t)p.max_pages * p.page_size, kUnit);
  L.bytes = L.logits + (weights ? (size_t)p.batch * n_q * L.logit_stride * 4 : 0);
  return L;
}

template <bool BF, int DP>
static int launch_attention(const AttnArgs& a, int grid, cudaStream_t st) {
  auto k = paged_attention_kernel<BF, DP>;
  const size_t smem = attn_smem<DP>(a.c.batch);
  // The attribute is the function's on the device, whoever sets it: always the
  // same value, what a block can have next to its static shared memory, so that
  // no thread lowers it under another's larger batch.
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
  k<<<grid, kThreads, smem, st>>>(a);
  TS_LAUNCH_CHECK();
  return TS_OK;
}

template <bool BF>
static int launch_attention(const AttnArgs& a, int grid, cudaStream_t st) {
  if (a.c.head_dim <= 64) return launch_attention<BF, 64>(a, grid, st);
  if (a.c.head_dim <= 128) return launch_attention<BF, 128>(a, grid, st);
  return launch_attention<BF, 256>(a, grid, st);
}

}  // namespace paged
}  // namespace ts

using namespace ts;
using namespace ts::paged;

extern "C" size_t ts_paged_attention_workspace_size(const ts_paged_cache* cache, int n_q, int accumulate) {
  if (cache == nullptr) return 0;
  return attn_layout(*cache, n_q, accumulate != 0).bytes;
}

extern "C" int ts_paged_decode_attention(const void* qkv, int64_t qkv_row_stride, int n_q, const ts_paged_cache* cache,
                                         const int64_t* positions, const float* rope_cos, const float* rope_sin,
                                         int64_t rope_rows, float scale, int accumulate, void* out,
                                         int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                                         void* stream) {
  AttnArgs a;
  const int rc = make_cache(cache, &a.c);
  if (rc != TS_OK) return rc;
  TS_REQUIRE(a.c.batch == 0 || (qkv && out), "NULL pointer");
  TS_REQUIRE((rope_cos == nullptr) == (rope_sin == nullptr), "rope_cos and rope_sin come both or neither");
  TS_REQUIRE(a.c.batch == 0 || positions != nullptr || (rope_cos == nullptr && a.c.slot_pos == nullptr),
             "positions are needed for the rotation and for slot_pos");
  TS_REQUIRE(n_q > 0 && n_q % a.c.n_kv == 0, "bad head counts");
  TS_REQUIRE(scale > 0.f && scale < INFINITY, "scale must be positive and finite");
  TS_REQUIRE(is_aligned(out, 4) && out_row_stride % 2 == 0, "rows of out must be 4-byte aligned");
  TS_REQUIRE(a.c.batch == 0 || !accumulate || a.c.scores != nullptr, "the cache has no scores to accumulate into");
  if (a.c.batch == 0) return TS_OK;
  a.group = n_q / a.c.n_kv;
  a.head_tiles = (a.group + kHeads - 1) / kHeads;
  TS_UNSUPPORTED((int64_t)a.c.batch * a.c.n_kv * a.head_tiles < (int64_t)kCounters, "too many heads in one call");
  TS_UNSUPPORTED(((int64_t)a.c.max_pages * a.c.page_size / kUnit + 1 + kRowCost) * a.c.batch * a.c.n_kv * a.head_tiles <
                     (int64_t)1 << 31,
                 "too many slots in one call");
  const Layout L = attn_layout(*cache, n_q, accumulate != 0);
  if (workspace == nullptr || workspace_bytes < L.bytes) {
    set_error("workspace of %zu bytes, %zu needed", workspace_bytes, L.bytes);
    return TS_ERR_WORKSPACE;
  }
  TS_REQUIRE(is_aligned(workspace, 16), "workspace must be 16-byte aligned");
  char* ws = reinterpret_cast<char*>(workspace);
  a.qkv = reinterpret_cast<const uint16_t*>(qkv);
  a.qkv_stride = qkv_row_stride;
  a.n_q = n_q;
  a.positions = positions;
  a.cos_t = rope_cos;
  a.sin_t = rope_sin;
  a.rope_rows = rope_rows;
  a.scale2 = scale * 1.4426950408889634f;
  a.out = reinterpret_cast<uint16_t*>(out);
  a.out_stride = out_row_stride;
  a.counters = reinterpret_cast<int*>(ws);
  a.partials = reinterpret_cast<float*>(ws + L.partials);
  a.lse2 = accumulate ? reinterpret_cast<float*>(ws + L.lse) : nullptr;
  a.logits = accumulate ? reinterpret_cast<float*>(ws + L.logits) : nullptr;
  a.logit_stride = L.logit_stride;
  a.page_shift = log2_of(a.c.page_size);
  a.one_page = a.c.page_size % kRows == 0 ? 1 : 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int grid = (int)grid_of(a.c.head_dim);
  const int r = cache->dtype == TS_BF16 ? launch_attention<true>(a, grid, st) : launch_attention<false>(a, grid, st);
  if (r != TS_OK || !accumulate) return r;
  const int rows = a.c.batch * a.c.n_kv;
  const int64_t cap = (int64_t)a.c.max_pages * a.c.page_size;
  const int per = a.c.page_size % 4 == 0 ? 4 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>((cap + 256 * per - 1) / (256 * per), (16 * sm_count() + rows - 1) / rows),
                     (unsigned)rows);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];                         // (it waits for the attention by itself)
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  TS_CUDA_TRY(per == 4 ? cudaLaunchKernelEx(&cfg, paged_weights_kernel<4>, a)
                       : cudaLaunchKernelEx(&cfg, paged_weights_kernel<1>, a));
  TS_LAUNCH_CHECK();
  return TS_OK;
}

extern "C" int ts_paged_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                               int tokens, const int32_t* n_new, const ts_paged_cache* cache, const int64_t* first,
                               const float* rope_cos, const float* rope_sin, int64_t rope_rows, const float* scores,
                               const int64_t* score_strides, void* stream) {
  AppendArgs a;
  const int rc = make_cache(cache, &a.c);
  if (rc != TS_OK) return rc;
  TS_REQUIRE(tokens >= 0, "bad tokens");
  if (a.c.batch == 0 || tokens == 0) return TS_OK;     // (there may be no memory behind the pointers)
  TS_REQUIRE(k && v && k_strides && v_strides, "NULL pointer");
  TS_REQUIRE((rope_cos == nullptr) == (rope_sin == nullptr), "rope_cos and rope_sin come both or neither");
  TS_REQUIRE(scores == nullptr || (a.c.scores != nullptr && score_strides != nullptr),
             "scores were given for a cache that keeps none");
  for (int i = 0; i < 3; ++i)
    TS_REQUIRE(k_strides[i] % 8 == 0 && v_strides[i] % 8 == 0, "k and v rows must be 16-byte aligned");
  TS_REQUIRE(is_aligned(k, 16) && is_aligned(v, 16), "k and v must be 16-byte aligned");
  a.k = reinterpret_cast<const uint16_t*>(k);
  a.v = reinterpret_cast<const uint16_t*>(v);
  a.kb = k_strides[0]; a.kt = k_strides[1]; a.kh = k_strides[2];
  a.vb = v_strides[0]; a.vt = v_strides[1]; a.vh = v_strides[2];
  a.first = first;
  a.n_new = n_new;
  a.tokens = tokens;
  a.cos_t = rope_cos;
  a.sin_t = rope_sin;
  a.rope_rows = rope_rows;
  a.scores = scores;
  a.sb = scores ? score_strides[0] : 0;
  a.sh = scores ? score_strides[1] : 0;
  a.st = scores ? score_strides[2] : 0;
  a.page_shift = log2_of(a.c.page_size);
  const int64_t items = (int64_t)((tokens + kTok - 1) / kTok) * a.c.n_kv;
  TS_UNSUPPORTED(a.c.batch <= 65535 && items < (int64_t)1 << 30, "too many sequences or tokens in one call");
  const dim3 grid((unsigned)std::max<int64_t>(1, std::min<int64_t>((items + 7) / 8, (16 * sm_count() + a.c.batch - 1) / a.c.batch)),
                  (unsigned)a.c.batch);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool rope = rope_cos != nullptr;
  if (cache->dtype == TS_BF16) {
    if (rope) paged_append_kernel<true, true><<<grid, 256, 0, st>>>(a);
    else paged_append_kernel<true, false><<<grid, 256, 0, st>>>(a);
  } else {
    if (rope) paged_append_kernel<false, true><<<grid, 256, 0, st>>>(a);
    else paged_append_kernel<false, false><<<grid, 256, 0, st>>>(a);
  }
  TS_LAUNCH_CHECK();
  return TS_OK;
}
