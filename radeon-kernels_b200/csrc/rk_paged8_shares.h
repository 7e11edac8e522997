// rk_paged8_shares.h -- how the decode attention over an 8-bit cache deals its work out to warps:
// whole numbers only, for the kernel (paged_attention8.cu) and for the host, which checks the
// bounds of what a warp may look up.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define RK_SHARES_FN __host__ __device__ __forceinline__
#else
#define RK_SHARES_FN inline
#endif

namespace rk {
namespace pa8 {

constexpr int WARPS = 4;  // of a CTA
// What starting and ending a range costs, in units (1 to 6 measured the same within 3 %: ragged batch 25.5
// to 25.8 us, 64 x 512 positions 23.1 to 24.0).
constexpr int RANGE_COST = 2;

// Positions of a unit, which is one tile of a warp.
RK_SHARES_FN constexpr int unit_of(int head_dim) { return head_dim == 256 ? 16 : 32; }

// Units of one (sequence, head tile); an empty sequence has one, which writes its NaN.
template <int D>
RK_SHARES_FN int units_of(int context) {
  return context <= unit_of(D) ? 1 : (context + unit_of(D) - 1) / unit_of(D);
}

// a / b for quotients below 2^21, where fp32 is off by one at most.
RK_SHARES_FN uint32_t quotient(uint32_t a, uint32_t b) {
#ifdef __CUDA_ARCH__
  uint32_t q = static_cast<uint32_t>(__fdividef(static_cast<float>(a), static_cast<float>(b)));
#else
  uint32_t q = static_cast<uint32_t>(static_cast<float>(a) / static_cast<float>(b));
#endif
  const int rest = static_cast<int>(a - q * b);
  if (rest < 0) --q;
  if (rest >= static_cast<int>(b)) ++q;
  return q;
}

// The shares of all warps: `extra` of them hold base + 1 places, the others base.  The host has
// checked that the places of the largest lengths fit 32 bits.
struct Shares {
  uint32_t total, warps, base, extra;
  RK_SHARES_FN void set(uint32_t places, uint32_t most_warps) {
    total = places;
    warps = most_warps < places ? most_warps : places;
    base = quotient(places, warps);
    extra = places - base * warps;
  }
  RK_SHARES_FN uint32_t start(uint32_t w) const { return w * base + (w < extra ? w : extra); }
  // The warp that holds a place.
  RK_SHARES_FN uint32_t owner(uint32_t place) const {
    const uint32_t wide = extra * (base + 1);
    const bool in = place < wide;
    return (in ? 0u : extra) + quotient(in ? place : place - wide, in ? base + 1 : base);
  }
};

// A place in the row of all units: sequence b, KV head h and its group hg of query heads (a
// head tile), unit c of its `units`; `left` units of a warp's share from here on.  Every range is
// followed by RANGE_COST places that hold no unit, so that shares with many short ranges hold fewer
// units.
struct Place {
  int b, h, hg, c, units, left;
};

// Whether the share holds a unit from here on.  One that holds none may have run past the last
// sequence -- a short share can begin behind the last range --, so nothing is looked up for it.
RK_SHARES_FN bool has_units(const Place& at) { return at.left > 0; }

// To the first unit of the next (sequence, head tile); returns whether that is another sequence,
// whose length the caller finds.
RK_SHARES_FN bool next_tile(Place& at, int kv_heads, int head_groups) {
  at.left -= at.units + RANGE_COST - at.c;
  at.c = 0;
  if (++at.hg < head_groups) return false;
  at.hg = 0;
  if (++at.h < kv_heads) return false;
  at.h = 0;
  ++at.b;
  return true;
}

// CTAs of a launch on a GPU that holds `most`: not more warps than units; RANGE_COST places of a
// range hold none.
RK_SHARES_FN int64_t ctas_of(int64_t ranges, int64_t units_per_range, int64_t most) {
  const int64_t warps = most * WARPS;
  if (ranges > warps || ranges * (units_per_range + RANGE_COST) >= warps) return most;
  return (ranges * (units_per_range + RANGE_COST) + WARPS - 1) / WARPS;
}

}  // namespace pa8
}  // namespace rk
