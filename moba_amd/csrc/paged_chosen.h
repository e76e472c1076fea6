// Rows that attend some blocks of their sequence's keys, each its own.
//
// A unit is up to 32 rows (tokens times heads) of one sequence and key/value head against a run of the keys of all blocks that at
// least one of them has chosen.  Its workgroup makes a list of these, in ascending order, with a bit for every row: a mask of rows for
// every block of the sequence, in LDS, a window at a time, into which the rows' entries are or-ed (whatever their order, one
// result), and of which the blocks with a row are counted through.  What a row has not chosen is masked, so that a block is read once
// however many rows have it.  The list's keys are numbered through (all of its blocks are whole but the last, which may be the
// sequence's last) and cut into as many runs as the batch's cut says, which knows only how many blocks the rows may have: about as many
// as if each had chosen its number at random.
//
// One token of 32 heads on 8, twelve blocks of 4096 behind 131072, 8 bits: 39 us and 4.8 for the merge, some 181 MB; sixteen users' tokens,
// sixteen blocks of 512, fp16: 47 and 4.6.  On one state, whose keys are partly in the last-level cache, the calls are 41.9 and 47.8; with a
// kernel before that makes the lists, and a cut by their lengths, 46.2 and 53.3; with a cut half way between rows that choose alike and
// at random 41.9 and 50.6; with more workgroups than fill the chip once 50 and 54 and more.
#pragma once
#include "attn_common.h"
#include "paged_cut.h"

namespace moba {

constexpr int kChosenRows = 32;    // of a unit
constexpr int kWindow = 4096;      // blocks whose masks lie in LDS at a time
constexpr int kLdsEntries = 1024;  // of a list that stays in LDS
constexpr int kListThreads = 256;

struct Chosen {
  int block;
  uint32_t rows;
};
struct ChosenTable : PageTable {
  const int32_t* blocks;  // [T, H, K], as they were given: any numbers
  Chosen* lists;          // [workgroups of a launch, room_of_list] for lists that may be longer than kLdsEntries, or null
  int K, each;            // entries of a row; pages of a block
  Divisor by_each;
  int room_of_list;
  int unit0, units;       // the first of this launch; of a launch
};
template <>
constexpr bool kChooses<ChosenTable> = true;

__device__ __forceinline__ int first_unit(const ChosenTable& t) { return t.unit0; }
__device__ __forceinline__ int block_keys(const ChosenTable& t) { return t.each << t.page_log2; }

__device__ __forceinline__ Chosen* list_of(const ChosenTable& t, char* lds) {
  return t.lists ? t.lists + (int64_t)blockIdx.x * t.room_of_list : reinterpret_cast<Chosen*>(lds);
}

// of blocks that `rows` rows have, K each at random
__device__ __forceinline__ float chosen_blocks(float blocks, float k, float rows) {
  return k < blocks ? blocks * (1.f - __builtin_amdgcn_exp2f(rows * __builtin_amdgcn_logf(1.f - k / blocks))) : blocks;
}
__device__ __forceinline__ Share share_of(const Shape<ChosenTable>& p, const Cut& c, const Sequence& s) {
  const int rows = (s.hi - s.lo) * p.rep, keys = keys_of(p, s);
  Share r = {s, 0, 0, 0};
  if (rows > 0 && keys > 0) {
    const int all = block_keys(p.table);
    const float some = chosen_blocks((float)((keys - 1) / all + 1), (float)p.table.K, (float)min(rows, kChosenRows)) * (float)all;
    r.tiles = (min(keys, (int)fminf(some + 0.5f, 2e9f)) - 1) / c.tile_keys + 1;
    r.groups = (rows - 1) / c.group_rows + 1;
  }
  return r;
}

// The list of a unit's rows row0 .. row0 + rows_here - 1, by the whole workgroup of kListThreads: the number of its keys.  `lds`: 4 * kWindow
// + 64 bytes; `list`: in LDS or memory.
__device__ __forceinline__ int make_list(const Shape<ChosenTable>& shape, const Sequence& seq, int hkv, int row0, int rows_here, char* lds,
                                         Chosen* list) {
  constexpr int kWaves = kListThreads / 64;
  uint32_t* const mask = reinterpret_cast<uint32_t*>(lds);
  volatile int* const sums = reinterpret_cast<volatile int*>(lds + 4 * kWindow);   // [kWaves], and the last block
  const ChosenTable& t = shape.table;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int keys = keys_of(shape, seq), all = block_keys(t), blocks = keys > 0 ? (keys - 1) / all + 1 : 0;
  int total = 0;
  for (int w0 = 0; w0 < blocks; w0 += kWindow) {
    const int here = min(kWindow, blocks - w0), each = (here + kListThreads - 1) / kListThreads;
    for (int i = tid; i < each * kListThreads; i += kListThreads) mask[i] = 0;
    __syncthreads();
    for (int i = tid; i < rows_here * t.K; i += kListThreads) {
      const int r = i / t.K, row = row0 + r, j = row / shape.rep;
      const int64_t position = seq.length - (seq.hi - seq.lo) + j;
      const int block = t.blocks[((int64_t)(seq.lo + j) * shape.H + hkv * shape.rep + row - j * shape.rep) * t.K + i - r * t.K];
      if (block >= w0 && block < w0 + here && (int64_t)block * all <= position) atomicOr(&mask[block - w0], 1u << r);
    }
    __syncthreads();
    // each thread its neighbouring blocks
    int mine = 0;
    for (int k = 0; k < each; ++k) mine += mask[tid * each + k] != 0;
    int upto = (int)upto_sum(mine);
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int found = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) upto += sums[w];
      found += sums[w];
    }
    int at = total + upto - mine;
    for (int k = 0; k < each; ++k) {
      const uint32_t who = mask[tid * each + k];
      if (!who) continue;
      list[at] = {w0 + tid * each + k, who};
      if (++at == total + found) sums[kWaves] = w0 + tid * each + k;
    }
    total += found;
    __syncthreads();   // (the list is written; masks and sums have been read)
  }
  if (total == 0) return 0;
  const int last = sums[kWaves];
  __syncthreads();   // (what comes next may lie here)
  return __builtin_amdgcn_readfirstlane((total - 1) * all + min(all, keys - last * all));
}

// Of key `key` of a list: its page's number in the sequence, the rows that have chosen it
__device__ __forceinline__ int chosen_page(const ChosenTable& t, const Chosen* list, int key, uint32_t& rows) {
  const int page = key >> t.page_log2, entry = quotient_or_same(page, t.by_each);
  const Chosen c = list[entry];
  rows = c.rows;
  return c.block * t.each + page - entry * t.each;
}

}  // namespace moba
