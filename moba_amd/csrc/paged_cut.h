// How the attention over the paged cache is cut into units of work, on the device.
//
// A unit is a group of query rows of one (sequence, key/value head) against a run of the sequence's keys.  The host knows
// neither the sequences' lengths nor how their new tokens are divided (both may change between replays of a captured
// call), so every workgroup finds its own unit: the runs are as long as fills the chip once with the whole batch's work,
// and the units of the sequences are counted through.  A long sequence among short ones gets the units that its keys ask for.
// One wave looks at 64 sequences at a time: up to 64 of them the whole cut is a load and a few dozen instructions.
#pragma once
#include "paged.h"

namespace moba {

// Of sequences with more than rows_over and at most rows_up_to query rows per key/value head:
struct Cut {
  int group_rows;  // query rows of a unit
  int tile_keys;   // a run of keys is a number of tiles
  int rows_over, rows_up_to;
  int target;      // units per key/value head that fill the chip
  int most;        // no more units per key/value head than this, whatever the batch
  int parts;       // no more than this of them where there is a sequence of several runs
};
constexpr int kWholeRun = 0x3fffffff;  // tiles
constexpr int kWholeAt = 4;  // with this many times `target` groups and more, a sequence's keys are one run

struct Shape {
  PageTable table;
  int H, Hkv, rep;
};

struct Share {
  int groups, tiles;  // of one sequence: groups of rows, tiles of keys (groups 0: not of this cut)
};
__device__ __forceinline__ int keys_of(const Shape& p, const Sequence& s) { return (int)min(s.length, room(p.table)); }
__device__ __forceinline__ Share share_of(const Shape& p, const Cut& c, const Sequence& s) {
  const int rows = (s.hi - s.lo) * p.rep;
  Share r;
  r.tiles = (keys_of(p, s) - 1) / c.tile_keys + 1;
  if (s.length == 0) r.tiles = 0;
  r.groups = rows > c.rows_over && rows <= c.rows_up_to && r.tiles > 0 ? (rows - 1) / c.group_rows + 1 : 0;
  return r;
}
__device__ __forceinline__ Share share_at(const Shape& p, const Cut& c, int b) {
  if (b >= p.table.B) return {0, 0};
  return share_of(p, c, sequence_of(p.table, b));
}

__device__ __forceinline__ int64_t wave_sum(int64_t x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

// Tiles of a run.  With work = sum of groups * tiles and n = sum of groups, runs of work / (target - n) tiles come to
// at most `target` units (each group's last run may be short); where the groups alone are more than half the target,
// runs of work / (target / 2), and where they fill the chip several times, whole sequences.
__device__ __forceinline__ int run_tiles(const Shape& p, const Cut& c, int lane, const Share& first) {
  int64_t work = 0, groups = 0;
  for (int b0 = 0; b0 < p.table.B; b0 += 64) {
    const Share s = b0 ? share_at(p, c, b0 + lane) : first;
    work += (int64_t)s.groups * s.tiles;
    groups += s.groups;
  }
  work = wave_sum(work);
  groups = wave_sum(groups);
  if (groups >= (int64_t)kWholeAt * c.target) return kWholeRun;
  const int64_t left = max(max((int64_t)c.target - groups, (int64_t)c.target / 2), (int64_t)1);
  return (int)min((work + left - 1) / left, (int64_t)kWholeRun);
}
__device__ __forceinline__ int runs_of(int tiles, int run) { return (tiles - 1) / run + 1; }

struct Unit {
  int b, group, run, runs, tiles;  // tiles: of the sequence
};
// unit number u: all groups of a sequence's first run, then of its second, ...  b = -1 past the last
__device__ __forceinline__ Unit unit_at(const Shape& p, const Cut& c, int u, int run, int lane, const Share& first) {
  int64_t base = 0;
  for (int b0 = 0; b0 < p.table.B; b0 += 64) {
    const Share s = b0 ? share_at(p, c, b0 + lane) : first;
    const int runs = s.groups ? runs_of(s.tiles, run) : 0;
    const int64_t mine = (int64_t)s.groups * runs;
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t below = __shfl_up(upto, o, 64);
      if (lane >= o) upto += below;
    }
    const uint64_t m = __ballot(base + upto > u);
    if (m) {
      const int at = __ffsll((unsigned long long)m) - 1;
      Unit r;
      r.b = b0 + at;
      r.runs = __shfl(runs, at, 64);
      r.tiles = __shfl(s.tiles, at, 64);
      const int groups = __shfl(s.groups, at, 64);
      const int rest = (int)(u - (base + __shfl(upto - mine, at, 64)));
      r.run = rest / groups;
      r.group = rest - r.run * groups;
      return r;
    }
    base += __shfl(upto, 63, 64);
  }
  return {-1, 0, 0, 0, 0};
}
// number of the first unit of sequence b
__device__ __forceinline__ int64_t first_unit(const Shape& p, const Cut& c, int b, int run, int lane, const Share& first) {
  int64_t n = 0;
  for (int b0 = 0; b0 < b; b0 += 64) {
    const Share s = b0 ? share_at(p, c, b0 + lane) : first;
    if (b0 + lane < b && s.groups) n += (int64_t)s.groups * runs_of(s.tiles, run);
  }
  return wave_sum(n);
}

}  // namespace moba
