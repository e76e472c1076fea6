// Sequences that begin with the same pages: what is common is attended once for all of them.
//
// cu_groups [G+1] cuts the sequences into groups of neighbours, shared [G] says how many leading tokens the tables of a group's
// sequences name the same pages for.  The batch is attended as G + B sequences: number g < G has all new tokens of group g as its
// rows and the first shared[g] tokens (rounded down to whole tiles) of the group's first table as its keys; number G + b has
// sequence b's rows and the keys behind those.  Every row sees keys up to its own position in either, so that the result is that
// of the sequences one by one, whatever `shared` says of equal tables.  A token's rows of both sides meet in the merge.
#pragma once
#include "paged_cut.h"

namespace moba {

constexpr int kSharedStep = 64;   // a run of keys begins at a multiple of this

struct SharedTable : PageTable {
  const int32_t* cu_groups;  // [G+1]
  const int32_t* shared;     // [G]
  int G;
};
template <>
constexpr bool kShares<SharedTable> = true;

__device__ __forceinline__ int first_member(const SharedTable& t, int g) { return min(max(t.cu_groups[g], 0), t.B); }
// the end of the keys that a group attends together
__device__ __forceinline__ int shared_keys(const SharedTable& t, int g) {
  return (int)min((int64_t)(max(t.shared[g], 0) & -kSharedStep), room(t));
}
// group of sequence b, -1 if it is in none: the last g < G with cu_groups[g] <= b, if b < cu_groups[g + 1]
__device__ __forceinline__ int group_of(const SharedTable& t, int b) {
  int lo = 0, hi = t.G;   // cu_groups[lo] <= b < cu_groups[hi], but for the ends
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.cu_groups[mid] <= b) lo = mid; else hi = mid;
  }
  return t.cu_groups[lo] <= b && b < t.cu_groups[lo + 1] ? lo : -1;
}

__device__ __forceinline__ int count_of(const SharedTable& t) { return t.G + t.B; }
__device__ __forceinline__ Sequence sequence_of(const SharedTable& t, int v) {
  Sequence s;
  if (v < t.G) {
    const int first = first_member(t, v), end = max(min(t.cu_groups[v + 1], t.B), first);
    s.lo = min(max(t.cu_new[first], 0), t.T);
    s.hi = min(max(t.cu_new[end], s.lo), t.T);
    s.length = shared_keys(t, v);
    s.begin = 0;
  } else {
    s = sequence_of(static_cast<const PageTable&>(t), v - t.G);
    const int g = group_of(t, v - t.G);
    s.begin = g >= 0 ? (int)min((int64_t)shared_keys(t, g), min(s.length, room(t))) : 0;
  }
  return s;
}

// Of sequence b, each lane its own, with the whole wave: groups and sequences that are 64 together at most are asked for at once, what they
// say of each other goes from lane to lane.
__device__ __forceinline__ Share share_at(const Shape<SharedTable>& p, const Cut& c, int b) {
  const SharedTable& t = p.table;
  if (count_of(t) > 64) {
    if (b >= count_of(t)) return {};
    Share r = share_of(p, c, sequence_of(t, b));
    r.row = b < t.G ? min(first_member(t, b), t.B - 1) : b - t.G;
    return r;
  }
  const bool group = b < t.G;
  const int first = t.cu_groups[min(b, t.G)], end = t.cu_groups[min(b + 1, t.G)], front = group ? shared_keys(t, b) : 0;
  Sequence s = sequence_of(static_cast<const PageTable&>(t), min(max(b - t.G, 0), t.B - 1));
  // a group's rows: from its first member's first to its last one's last
  const int m0 = min(max(first, 0), t.B), m1 = max(min(end, t.B), m0);
  const int lo = __shfl(s.lo, t.G + min(m0, t.B - 1), 64), hi = __shfl(s.hi, t.G + max(m1 - 1, 0), 64);
  // a sequence's group: the last that begins no later
  int g = 0;
  for (int above = t.G; __any(above - g > 1);) {
    const int mid = (g + above) >> 1, begins = __shfl(first, mid, 64);
    if (above - g > 1) {
      if (begins <= b - t.G) g = mid; else above = mid;
    }
  }
  const int g_first = __shfl(first, g, 64), g_end = __shfl(end, g, 64), g_front = __shfl(front, g, 64);
  if (b >= count_of(t)) return {};
  if (group) {
    s = {lo, m1 > m0 ? max(hi, lo) : lo, front, 0};
  } else {
    s.begin = g_first <= b - t.G && b - t.G < g_end ? (int)min((int64_t)g_front, min(s.length, room(t))) : 0;
  }
  Share r = share_of(p, c, s);
  r.row = group ? min(m0, t.B - 1) : b - t.G;
  return r;
}

// Position of new token j of a unit's rows: in its own sequence, the last that begins no later.  With the whole wave, whose lanes have
// groups and sequences that are 64 together at most.
__device__ __forceinline__ int position_at(const SharedTable& t, const Unit& u, int j, const Sequence& mine) {
  if (u.b >= t.G) return (int)u.seq.length - (u.seq.hi - u.seq.lo) + j;
  const int token = u.seq.lo + j;
  if (count_of(t) <= 64) {
    int lo = 0;
    for (int above = t.B; __any(above - lo > 1);) {
      const int mid = (lo + above) >> 1, begins = __shfl(mine.lo, t.G + mid, 64);
      if (above - lo > 1) {
        if (begins <= token) lo = mid; else above = mid;
      }
    }
    const int ends = __shfl(mine.hi, t.G + lo, 64), length = __shfl((int)mine.length, t.G + lo, 64);
    return (int)min((int64_t)length - ends + token, (int64_t)0x7fffffff);
  }
  const int first = first_member(t, u.b), end = min(t.cu_groups[u.b + 1], t.B);
  int lo = 0, hi = end - first;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.cu_new[first + mid] <= token) lo = mid; else hi = mid;
  }
  const Sequence s = sequence_of(static_cast<const PageTable&>(t), min(first + lo, t.B - 1));
  return (int)min(s.length - s.hi + token, (int64_t)0x7fffffff);
}
// (a group's rows are of several sequences)
__device__ __forceinline__ int least_position(const SharedTable& t, const Unit& u, int first, int position) {
  if (u.b >= t.G) return position_at(t, u, first, u.seq);
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) position = min(position, __shfl_xor(position, d, 64));
  return __builtin_amdgcn_readfirstlane(position);
}
__device__ __forceinline__ int last_seen(const SharedTable& t, const Unit& u, int j) {
  return u.b >= t.G ? position_at(t, u, j, u.seq) : 0x7ffffffe;
}

}  // namespace moba
