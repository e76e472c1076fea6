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
  bool even;       // kShares: runs by even_run()
};
constexpr int kWholeRun = 0x3fffffff;  // tiles
// With this many times `target` groups and more, a sequence's keys are one run.  That is right for sequences of like lengths, and slow for one
// long one among them: one token each for 255 sequences, 131072 keys and 254 of 513, 8 heads, 8 bits: 120 us; one more of these: 1135.
constexpr int kWholeAt = 4;

// Table: PageTable, or another that has its own of the functions below, and kShares or kChooses
template <class Table>
struct Shape {
  Table table;
  int H, Hkv, rep;
};
__device__ __forceinline__ int count_of(const PageTable& t) { return t.B; }                // sequences
__device__ __forceinline__ int first_unit(const PageTable&) { return 0; }                  // of a launch
template <class Table>
constexpr bool kShares = false;   // whether a token attends keys of more than one sequence
template <class Table>
constexpr bool kChooses = false;  // whether a row attends some of the keys only

// A sequence's part in a cut: groups of rows (0: none of its units are of this cut), tiles of keys; kShares: its row of the page table
struct Share {
  Sequence seq;
  int groups, tiles, row;
};
// the end of a sequence's keys
template <class Table>
__device__ __forceinline__ int keys_of(const Shape<Table>& p, const Sequence& s) { return (int)min(s.length, room(p.table)); }
template <class Table>
__device__ __forceinline__ Share share_of(const Shape<Table>& p, const Cut& c, const Sequence& s) {
  const int rows = (s.hi - s.lo) * p.rep, keys = keys_of(p, s) - s.begin;
  Share r = {};
  r.seq = s;
  r.tiles = keys > 0 ? (keys - 1) / c.tile_keys + 1 : 0;
  r.groups = rows > c.rows_over && rows <= c.rows_up_to && keys > 0 ? (rows - 1) / c.group_rows + 1 : 0;
  return r;
}
// of sequence b, each lane its own
template <class Table>
__device__ __forceinline__ Share share_at(const Shape<Table>& p, const Cut& c, int b) {
  if (b >= count_of(p.table)) return {};
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

// (a whole-number division is some forty instructions; this is exact up to 2^22 tiles, more go that way)
__device__ __forceinline__ int runs_of(int tiles, int run) {
  if (__any(tiles > 1 << 22)) return (tiles - 1) / run + 1;
  int n = (int)((float)(tiles - 1) * __builtin_amdgcn_rcpf((float)run));
  n += (n + 1) * run <= tiles - 1;
  return n - (n * run > tiles - 1) + 1;
}

// the largest of the lanes' x, none of them negative
__device__ __forceinline__ int wave_max(int x) {
#define MOBA_DPP_MAX(ctrl, rows) x = max(x, __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, false))
  MOBA_DPP_MAX(0x111, 0xf);
  MOBA_DPP_MAX(0x112, 0xf);
  MOBA_DPP_MAX(0x114, 0xf);
  MOBA_DPP_MAX(0x118, 0xf);
  MOBA_DPP_MAX(0x142, 0xa);
  MOBA_DPP_MAX(0x143, 0xc);
#undef MOBA_DPP_MAX
  return __builtin_amdgcn_readlane(x, 63);
}

// Tiles of a run where units are long and of many lengths: a small part of the longest sequence, each lane its own, such that the rounds of
// the long units, and all units shared out evenly, take least; a unit's start counts as least_tiles.  (Up to 64 sequences; `otherwise` where
// every choice is more units than are launched.)  700 and 500 tokens behind 12288 shared ones, 8 heads: 8 bits 317 us, 349 with the runs of
// run_tiles(); 16 bits 314 and 380; 4 times 64 behind 30000 153 and 148.
__device__ __forceinline__ int even_run(const Cut& c, int lane, const Share& first, int sequences, int64_t work, int otherwise) {
  constexpr int kParts = 32;
  const int longest = wave_max(first.groups ? first.tiles : 0), run = max((longest - 1) / (min(lane, kParts - 1) + 1) + 1, c.least_tiles);
  int units = 0, long_units = 0;
  for (int b = 0; b < sequences; ++b) {
    const int groups = __builtin_amdgcn_readlane(first.groups, b), tiles = __builtin_amdgcn_readlane(first.tiles, b);
    if (groups == 0) continue;
    const int runs = runs_of(tiles, run);
    units += groups * runs;
    long_units += 2 * tiles > run * runs ? groups * runs : 0;
  }
  const float rounds = (float)((long_units - 1) / c.target + 1) * (float)(run + c.least_tiles);
  const float even = ((float)work + (float)units * (float)c.least_tiles) / (float)c.target;
  float cost = units <= c.most ? fmaxf(rounds, even) : 1e30f;
  const float mine = cost;
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) cost = fminf(cost, __shfl_xor(cost, d, 64));
  const int at = __ffsll((unsigned long long)__ballot(mine == cost)) - 1;
  return cost < 1e30f ? __builtin_amdgcn_readlane(run, at) : otherwise;
}

// Tiles of a run.  With work = sum of groups * tiles and n = sum of groups: the shortest runs, of work / target tiles or some
// more, that come to at most `target` units (each group's last run may be short); runs of work / (target - n) always do.  Where the groups
// alone are more than half the target, of work / (target / 2), and where they fill the chip several times, whole sequences.  No runs of
// fewer than least_tiles: where a unit's start outweighs a tile, short runs cost more in the merge than they save.
template <class Table>
__device__ __forceinline__ int run_tiles(const Shape<Table>& p, const Cut& c, int lane, const Share& first) {
  int64_t work = 0, groups = 0;
  for (int b0 = 0; b0 < count_of(p.table); b0 += 64) {
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
  if constexpr (kShares<Table>) {
    if (c.even && groups > 0 && count_of(p.table) <= 64 && work < 1LL << 24) return even_run(c, lane, first, count_of(p.table), work, safe);
  }
  if (count_of(p.table) <= 64 && groups <= c.target)
    for (int run = max(ceil_div(work, c.target), c.least_tiles); run < safe; run += run / 16 + 1)
      if (wave_sum(first.groups ? first.groups * runs_of(first.tiles, run) : 0) <= (uint32_t)c.target) return run;
  return safe;
}

struct Unit {
  Sequence seq;
  int b, row, group, run, runs, groups, tiles, first;  // row: of the page table; tiles: of the sequence; first: number of the sequence's first unit
};
// unit number u: all groups of a sequence's first run, then of its second, ...; b = -1 past the last.  kShares, up to 64 sequences: those
// with long runs first, so that none of these is left for the end (pieces of 200, 300, 301 and 97 tokens behind 12288 shared ones: 315 us
// otherwise, 243 so; shorter steps between the lengths gain nothing, as workgroups start in the order of their numbers).
template <class Table>
__device__ __forceinline__ Unit unit_at(const Shape<Table>& p, const Cut& c, int u, int run, int lane, const Share& first) {
  int64_t base = 0;
  for (int b0 = 0; b0 < count_of(p.table); b0 += 64) {
    const Share s = b0 ? share_at(p, c, b0 + lane) : first;
    const int runs = s.groups ? runs_of(s.tiles, run) : 0;
    const uint32_t mine = (uint32_t)s.groups * runs;
    uint32_t upto = upto_sum(mine), all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    if constexpr (kShares<Table>) {
      if (count_of(p.table) <= 64) {
        const int per = runs ? (s.tiles - 1) / runs + 1 : 0;
        const bool is_long = 2 * per > wave_max(per);
        const uint32_t upto_long = upto_sum(is_long ? mine : 0), longs = (uint32_t)__builtin_amdgcn_readlane((int)upto_long, 63);
        upto = is_long ? upto_long : longs + upto - upto_long;
      }
    }
    const uint64_t m = __ballot(base + upto > u && base + upto - mine <= u && mine > 0);
    if (m) {
      const int at = __ffsll((unsigned long long)m) - 1;
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
      Unit r;
      r.b = b0 + at;
      r.row = kShares<Table> ? of(s.row) : r.b;
      r.seq.lo = of(s.seq.lo);
      r.seq.hi = of(s.seq.hi);
      r.seq.length = of((int)s.seq.length);
      r.seq.begin = kShares<Table> ? of(s.seq.begin) : 0;
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
    base += all;
  }
  Unit none = {};
  none.b = -1;
  return none;
}

// The unit of a workgroup, its key/value head, and the number under which it leaves what the merge has to know; false: none.  Workgroups
// are numbered by unit and head.  first: share_at() of the lanes.
template <class Table>
__device__ __forceinline__ bool find_unit(const Shape<Table>& p, const Cut& c, int lane, Unit& unit, int& hkv, int& item, Share& first) {
  const int at = (int)blockIdx.x / p.Hkv, u = first_unit(p.table) + at;
  hkv = (int)blockIdx.x - at * p.Hkv;
  first = share_at(p, c, lane);
  const int run = run_tiles(p, c, lane, first);
  if (run == 0) return false;   // (no work at all)
  unit = unit_at(p, c, u, run, lane, first);
  item = unit.b;
  return unit.b >= 0 && (unit.runs == 1 || u < c.parts);   // (the latter: row ranges that are none)
}

// What the merge has to know of a sequence, left for it by the sequence's first unit
struct Runs {
  int first, runs, groups;
};

}  // namespace moba
