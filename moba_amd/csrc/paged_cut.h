// How the attention over the paged cache is cut into units of work, on the device.
//
// A unit is a group of query rows of one (sequence, key/value head) against a run of the sequence's keys.  The host knows
// neither the sequences' lengths nor how their new tokens are divided (both may change between replays of a captured
// call), so every workgroup finds its own unit, and the units of the sequences are counted through.  Up to as many groups as the
// chip has places (half as many where there are more than 64 sequences), the runs are as long as fills the chip once with the
// whole batch's work, so that a long sequence among short ones gets the units that its keys ask for.  With more they are the work
// of two places each, however full the last round is, and from kWholeAt times as many on a sequence's keys are one run.  Every
// group counts with all of its sequence's keys, those that no row of it sees included.
// One wave looks at 64 sequences at a time: up to 64 of them the whole cut is one load and some hundred cycles.
#pragma once
#include "paged.h"

namespace moba {

// Of sequences with more than rows_over and at most rows_up_to query rows per key/value head:
struct Cut {
  int group_rows;  // query rows of a unit
  int tile_keys;   // a run of keys is a number of tiles,
  int least_tiles; // no fewer than this
  int rows_over, rows_up_to;
  int target;      // units per key/value head that fill the chip
  int most;        // no more units per key/value head than this, whatever the batch
  int parts;       // no more than this of them where there is a sequence of several runs
};
constexpr int kWholeRun = 0x3fffffff;  // tiles
// With this many times `target` groups and more, a sequence's keys are one run.  That is right for sequences of like lengths, and slow for one
// long one among them: one token each for 255 sequences, 131072 keys and 254 of 513, 8 heads, 8 bits: 120 us; one more of these: 1135.
constexpr int kWholeAt = 4;

struct Shape {
  PageTable table;
  int H, Hkv, rep;
};

// A sequence's part in a cut: groups of rows (0: none of its units are of this cut), tiles of keys
struct Share {
  Sequence seq;
  int groups, tiles;
};
__device__ __forceinline__ int keys_of(const Shape& p, const Sequence& s) { return (int)min(s.length, room(p.table)); }
__device__ __forceinline__ Share share_of(const Shape& p, const Cut& c, const Sequence& s) {
  const int rows = (s.hi - s.lo) * p.rep, keys = keys_of(p, s);
  Share r;
  r.seq = s;
  r.tiles = keys > 0 ? (keys - 1) / c.tile_keys + 1 : 0;
  r.groups = rows > c.rows_over && rows <= c.rows_up_to && keys > 0 ? (rows - 1) / c.group_rows + 1 : 0;
  return r;
}
// of sequence b, each lane its own
__device__ __forceinline__ Share share_at(const Shape& p, const Cut& c, int b) {
  if (b >= p.table.B) return {{0, 0, 0}, 0, 0};
  return share_of(p, c, sequence_of(p.table, b));
}

// sum of x over the lanes up to this one (wrapping)
__device__ __forceinline__ uint32_t upto_sum(uint32_t x) {
#define MOBA_DPP_ADD(ctrl, rows) x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, false)
  MOBA_DPP_ADD(0x111, 0xf);  // from 1, 2, 4, 8 lanes below in the row of 16
  MOBA_DPP_ADD(0x112, 0xf);
  MOBA_DPP_ADD(0x114, 0xf);
  MOBA_DPP_ADD(0x118, 0xf);
  MOBA_DPP_ADD(0x142, 0xa);  // a row's last lane to the row above
  MOBA_DPP_ADD(0x143, 0xc);  // lane 31 to the upper half
#undef MOBA_DPP_ADD
  return x;
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)upto_sum(x), 63); }

__device__ __forceinline__ int runs_of(int tiles, int run) { return (tiles - 1) / run + 1; }

// Tiles of a run.  With work = sum of groups * tiles and n = sum of groups: the shortest runs, of work / target tiles or some
// more, that come to at most `target` units (each group's last run may be short); runs of work / (target - n) always do.  Where the groups
// alone are more than half the target, of work / (target / 2), and where they fill the chip several times, whole sequences.  No runs of
// fewer than least_tiles: where a unit's start outweighs a tile, short runs cost more in the merge than they save.
__device__ __forceinline__ int run_tiles(const Shape& p, const Cut& c, int lane, const Share& first) {
  int64_t work = 0, groups = 0;
  for (int b0 = 0; b0 < p.table.B; b0 += 64) {
    const Share s = b0 ? share_at(p, c, b0 + lane) : first;
    const int64_t w = (int64_t)s.groups * s.tiles;   // (below 2^56: in pieces of 24 bits a wave's sum fits 32)
    work += wave_sum((uint32_t)w & 0xffffff) + ((int64_t)wave_sum((uint32_t)(w >> 24) & 0xffffff) << 24) +
            ((int64_t)wave_sum((uint32_t)(w >> 48)) << 48);
    groups += wave_sum(s.groups);
  }
  if (groups >= (int64_t)kWholeAt * c.target) return kWholeRun;
  auto ceil_div = [](int64_t a, int64_t b) {   // (64-bit division is slow)
    return a < 1LL << 31 ? (int)(((uint32_t)a + (uint32_t)b - 1) / (uint32_t)b) : (int)min((a + b - 1) / b, (int64_t)kWholeRun);
  };
  const int safe = max(ceil_div(work, max(max((int64_t)c.target - groups, (int64_t)c.target / 2), (int64_t)1)), work > 0 ? c.least_tiles : 0);
  if (p.table.B <= 64 && groups <= c.target)
    for (int run = max(ceil_div(work, c.target), c.least_tiles); run < safe; run += run / 16 + 1)
      if (wave_sum(first.groups ? first.groups * runs_of(first.tiles, run) : 0) <= (uint32_t)c.target) return run;
  return safe;
}

struct Unit {
  Sequence seq;
  int b, group, run, runs, groups, tiles, first;  // tiles: of the sequence; first: number of the sequence's first unit
};
// unit number u: all groups of a sequence's first run, then of its second, ...  b = -1 past the last
__device__ __forceinline__ Unit unit_at(const Shape& p, const Cut& c, int u, int run, int lane, const Share& first) {
  int64_t base = 0;
  for (int b0 = 0; b0 < p.table.B; b0 += 64) {
    const Share s = b0 ? share_at(p, c, b0 + lane) : first;
    const int runs = s.groups ? runs_of(s.tiles, run) : 0;
    const uint32_t mine = (uint32_t)s.groups * runs, upto = upto_sum(mine);
    const uint64_t m = __ballot(base + upto > u && mine > 0);
    if (m) {
      const int at = __ffsll((unsigned long long)m) - 1;
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
      Unit r;
      r.b = b0 + at;
      r.seq.lo = of(s.seq.lo);
      r.seq.hi = of(s.seq.hi);
      r.seq.length = of((int)s.seq.length);
      r.runs = of(runs);
      r.groups = of(s.groups);
      r.tiles = of(s.tiles);
      r.first = (int)(base + (uint32_t)of((int)(upto - mine)));
      const int rest = u - r.first;
      r.run = rest / r.groups;
      r.group = rest - r.run * r.groups;
      if (rest < 0 || r.run >= r.runs) r.b = -1;   // (row ranges that are none: more units than 32 bits number)
      return r;
    }
    base += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
  }
  Unit none = {};
  none.b = -1;
  return none;
}

// What the merge has to know of a sequence, left for it by the sequence's first unit
struct Runs {
  int first, runs, groups;
};

}  // namespace moba
