// Rows that attend some blocks of their sequence's keys, each its own: how the blocks become units of work.
//
// A unit is up to 32 rows (tokens times heads) of one sequence and key/value head against a run of the keys of all blocks that at
// least one of them has chosen: a list, in ascending order, of blocks with a bit for every row.  What a row has not chosen is masked, so
// that a block is read once however many rows have it.  The list's keys are numbered through (all of its blocks are
// whole but the last, which may be the sequence's last), and cut into runs as the whole keys of a sequence are (paged_cut.h).
#pragma once
#include "attn_common.h"
#include "paged_cut.h"

namespace moba {

constexpr int kChosenRows = 32;   // of a unit

struct Chosen {
  int block;
  uint32_t rows;
};
struct ChosenTable : PageTable {
  const int32_t* blocks;  // [T, H, K], as they were given: any numbers
  const Chosen* lists;    // [items, room_of_list]
  const int32_t* keys;    // [items]: keys of the list's blocks
  int K, each;            // entries of a row; pages of a block
  Divisor by_each;
  int room_of_list, items, target;  // items: (group of rows, key/value head), by the batch's bounds
};
template <>
constexpr bool kChooses<ChosenTable> = true;

// Groups of rows of the sequences, counted so that a sequence's first follows from where its rows begin (some numbers are nobody's):
// sequence b's first is this many rows * rep / 32 + b
__device__ __forceinline__ int64_t first_group(int lo, int rep, int b) { return (int64_t)lo * rep / kChosenRows + b; }

// The unit of a workgroup.  Runs as in run_tiles() and unit_at(), over items instead of sequences; with kWholeAt times as many items
// as fill the chip an item's keys are one run.
__device__ __forceinline__ bool find_unit(const Shape<ChosenTable>& shape, const Cut& c, int lane, Unit& unit, int& hkv, int& item) {
  const ChosenTable& t = shape.table;
  const int u = blockIdx.x;
  unit = {};
  auto tiles_of = [&](int i) { return i < t.items ? (t.keys[i] + c.tile_keys - 1) / c.tile_keys : 0; };
  if (t.items >= kWholeAt * t.target) {
    item = u;
    unit.tiles = __builtin_amdgcn_readfirstlane(tiles_of(u));
    unit.runs = 1;
    unit.first = u;
  } else {
    constexpr int kKept = 8;   // of the items' tiles, 64 at a time
    int kept[kKept];
    int64_t work = 0;
    int groups = 0;
#pragma unroll
    for (int k = 0; k < kKept; ++k) kept[k] = tiles_of(64 * k + lane);
#pragma unroll
    for (int k = 0; k < kKept; ++k) {
      work += wave_sum(kept[k]);
      groups += __builtin_popcountll(__ballot(kept[k] > 0));
    }
    for (int i0 = 64 * kKept; i0 < t.items; i0 += 64) {
      const int tiles = tiles_of(i0 + lane);
      work += wave_sum(tiles);
      groups += __builtin_popcountll(__ballot(tiles > 0));
    }
    const int places = max(max(t.target - groups, t.target / 2), 1);
    int run = max((int)min((work + places - 1) / places, (int64_t)kWholeRun), c.least_tiles);
    if (t.items <= 64 * kKept && groups <= t.target) {   // the shortest runs that fit
      const int safe = run;
      for (int r = max((int)min((work + t.target - 1) / t.target, (int64_t)kWholeRun), c.least_tiles); r < safe; r += r / 16 + 1) {
        int n = 0;
#pragma unroll
        for (int k = 0; k < kKept; ++k) n += kept[k] ? runs_of(kept[k], r) : 0;
        if (wave_sum(n) <= (uint32_t)t.target) {
          run = r;
          break;
        }
      }
    }
    int base = 0;
    item = -1;
    auto look = [&](int i0, int tiles) __attribute__((always_inline)) {
      const int runs = tiles ? runs_of(tiles, run) : 0, upto = (int)upto_sum(runs);
      const uint64_t m = __ballot(base + upto > u && runs > 0);
      if (m && item < 0) {
        const int at = __ffsll((unsigned long long)m) - 1;
        item = i0 + at;
        unit.tiles = __builtin_amdgcn_readlane(tiles, at);
        unit.runs = __builtin_amdgcn_readlane(runs, at);
        unit.first = base + __builtin_amdgcn_readlane(upto - runs, at);
        unit.run = u - unit.first;
      }
      base += __builtin_amdgcn_readlane(upto, 63);
    };
#pragma unroll
    for (int k = 0; k < kKept; ++k) look(64 * k, kept[k]);
    for (int i0 = 64 * kKept; i0 < t.items && item < 0; i0 += 64) look(i0, tiles_of(i0 + lane));
  }
  if (item < 0 || unit.tiles == 0) return false;
  const int g = item / shape.Hkv;
  hkv = item - g * shape.Hkv;
  unit.b = last_up_to(t, g, lane, unit.seq, [&](int b, int lo) { return first_group(lo, shape.rep, b); });
  if (unit.b < 0) return false;
  unit.group = (int)(g - first_group(unit.seq.lo, shape.rep, unit.b));
  unit.groups = 1;
  return unit.group >= 0 && unit.group * kChosenRows < (unit.seq.hi - unit.seq.lo) * shape.rep;
}

// Of key `key` of an item's list: its page's number in the sequence, the rows that have chosen it
__device__ __forceinline__ int chosen_page(const ChosenTable& t, int item, int key, uint32_t& rows) {
  const int page = key >> t.page_log2, entry = quotient_or_same(page, t.by_each);
  const Chosen c = t.lists[(int64_t)item * t.room_of_list + entry];
  rows = c.rows;
  return c.block * t.each + page - entry * t.each;
}

}  // namespace moba
