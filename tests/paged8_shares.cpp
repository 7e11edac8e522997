// The arithmetic by which the 8-bit decode attention deals its work out, on the host: what every warp of
// a launch begins with and walks over.
#include "rk_paged8_shares.h"

using namespace rk::pa8;

template <int D>
static int64_t walks(const int* lengths, int batch, int kv_heads, int head_groups, int64_t ctas, int64_t* first,
                     int32_t* visits, int64_t most) {
  const int tiles = kv_heads * head_groups;
  uint32_t total = 0;
  for (int b = 0; b < batch; ++b) total += (units_of<D>(lengths[b]) + RANGE_COST) * tiles;
  const uint32_t warps = static_cast<uint32_t>(ctas * WARPS);
  Shares shares;
  shares.set(total, warps);
  int64_t n = 0;
  for (uint32_t me = 0; me < warps; ++me) {
    const bool idle = me >= shares.warps;
    const uint32_t u0 = shares.start(idle ? 0 : me);
    Place at{};
    at.left = idle ? 0 : static_cast<int>(shares.start(me + 1) - u0);
    uint32_t before = 0;
    for (;; ++at.b) {
      at.units = units_of<D>(lengths[at.b]);
      const uint32_t places = (at.units + RANGE_COST) * tiles;
      if (before + places > u0) break;
      before += places;
    }
    const int tile = static_cast<int>(quotient(u0 - before, at.units + RANGE_COST));
    at.c = static_cast<int>(u0 - before) - tile * (at.units + RANGE_COST);
    at.h = tile / head_groups;
    at.hg = tile - at.h * head_groups;
    const auto next = [&] {
      if (next_tile(at, kv_heads, head_groups)) at.units = units_of<D>(lengths[at.b < batch ? at.b : batch - 1]);
    };
    if (at.c >= at.units) next();
    // The sequence that the warp begins with, and whether it looks anything up for it.
    first[2 * me] = at.b;
    first[2 * me + 1] = has_units(at) ? 1 : 0;
    while (has_units(at)) {
      if (n == most) return -1;
      const int32_t visit[5] = {static_cast<int32_t>(me), at.b, at.h, at.hg, at.c};
      for (int i = 0; i < 5; ++i) visits[5 * n + i] = visit[i];
      ++n;
      ++at.c;
      --at.left;
      if (at.c == at.units) next();
    }
  }
  return n;
}

extern "C" {
int64_t shares_ctas(int64_t ranges, int64_t units_per_range, int64_t most) { return ctas_of(ranges, units_per_range, most); }
int shares_warps() { return WARPS; }
int shares_unit(int head_dim) { return unit_of(head_dim); }

// Every unit that a warp takes, as (warp, sequence, KV head, head group, unit) in `visits`; returns how many.
// `first`: [ctas * WARPS][2].
int64_t shares_walks(const int* lengths, int batch, int kv_heads, int head_groups, int head_dim, int64_t ctas, int64_t* first,
                     int32_t* visits, int64_t most) {
  return head_dim == 256 ? walks<256>(lengths, batch, kv_heads, head_groups, ctas, first, visits, most)
                         : walks<128>(lengths, batch, kv_heads, head_groups, ctas, first, visits, most);
}
}
