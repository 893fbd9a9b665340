// How the attention kernels over the paged cache cut their work: units of a kv head's
// slots, dealt out to CTAs, a quarter of each unit to a warp (64 slots and 16 in the 16-bit
// kernel, whose constants stand here, 128 and 32 in the 8-bit one); and the matrix
// instructions that both use.
#pragma once

#include "paged.cuh"

namespace ts {
namespace paged {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;                  // slots of a warp's share of a unit
constexpr int kUnit = kWarps * kRows;      // slots of a unit
constexpr unsigned kUnitCost = 1800;       // cycles of a unit, see choose_deal
constexpr int kRowCost = 6;                // units that starting and joining a row costs
constexpr int kFullUnits = 8;              // units per CTA from which that cost is counted
constexpr int kMaxPieces = 96;             // CTAs that share a kv head's units at most

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <bool BF>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};" : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};" : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Equal shares of `total` units for n CTAs: the first total % n get one more.
struct Shares {
  unsigned q, r;
  __device__ __forceinline__ Shares(unsigned total, unsigned n) : q(total / n), r(total - total / n * n) {}
  __device__ __forceinline__ unsigned begin(unsigned i) const { return i * q + min(i, r); }
  __device__ __forceinline__ unsigned owner(unsigned u) const {
    return u < r * (q + 1) ? u / (q + 1) : r + (u - r * (q + 1)) / q;
  }
};

// How the rows' units (a row: a kv head's, or 16 of its query heads) are dealt
// out to CTAs.
struct Deal {
  int front;          // see below
  unsigned n_cta;
};

// Cycles, as measured in the 16-bit kernel where CTAs have little to do: a unit 1800; a row's start
// and its warps' join 6000; the join of pieces 3000, and for each eight query
// heads 2500 and 1200 for each eight pieces. The 8-bit kernel takes the same numbers for its own units,
// which have as many bytes. (A whole warp calls it.)
__device__ __forceinline__ Deal choose_deal(unsigned units, unsigned rows, int longest, unsigned grid, int heads) {
  if (rows == 0) return {0, 0};
  const unsigned turns = (heads + 2 * kWarps - 1) / (2 * kWarps);
  auto join = [&](unsigned pieces) { return pieces > 1 ? 3000 + turns * (2500 + (pieces + 7) / 8 * 1200) : 0; };
  // Equal shares of all units laid end to end, each row with a few units in
  // front of its own for its start, so that a CTA of many short rows gets
  // fewer units than one of few long ones. No row in more than kMaxPieces + 1.
  const bool full = units >= kFullUnits * grid || rows > grid;
  Deal d;
  d.front = full ? kRowCost : 0;
  const unsigned total = units + rows * d.front;
  const unsigned least = max((unsigned)d.front + 1, (longest + d.front + kMaxPieces - 1) / kMaxPieces);
  d.n_cta = max(1u, min(grid, total / least));
  if (full) return d;
  // Where a launch has few units: each row in equal parts of CTAs of its own,
  // if that lets the last of them finish sooner.
  const unsigned share = (units + d.n_cta - 1) / d.n_cta;
  const unsigned shares_cost = share * kUnitCost + (rows > 1 ? 6000 : 0) + join((longest + share - 1) / share + 1);
  // lane i looks at i + 1 and at 34 + 2 i parts
  unsigned best = 0xFFFFFFFFu;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const unsigned p = k == 0 ? (threadIdx.x & 31) + 1 : 34 + 2 * (threadIdx.x & 31);
    const unsigned q = (longest + p - 1) / p;
    if (p <= (unsigned)min(longest, kMaxPieces) && rows * p <= grid) best = min(best, (q * kUnitCost + join(p)) << 7 | p);
  }
  best = __reduce_min_sync(0xffffffffu, best);
  if (best >> 7 < shares_cost) {
    const unsigned p = best & 127;
    d.front = -(int)((longest + p - 1) / p * p);
    d.n_cta = rows * p;
  }
  return d;
}

}  // namespace paged
}  // namespace ts
