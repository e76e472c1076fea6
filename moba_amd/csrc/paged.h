// The paged key/value cache: what its kernels share.
//
// A page holds page_size tokens (a power of two from 16 to 256) of all key/value heads: pages [num_pages, Hkv, page_size, D], so
// that the tokens of a (page, head) are contiguous: whole cache lines for the attention, which reads one head at a time.
// Elements are those of the model (16 bits), or e4m3 with a 32-bit scale for every (page, head) of the keys and of the
// values: an element stands for its value times its page's scale.
// page_table [B, max_pages] names the pages of every sequence; lengths [B] counts its tokens, the new ones included; cu_new
// [B+1] delimits each sequence's new tokens among the packed rows of q, k, v.  All three are read on the device: a call
// depends on no host copy of them, and a captured one follows them.  Nothing in them is trusted: whatever they hold, no access leaves
// the tensors (a page id out of range is a page without keys; lengths and row ranges are cut to what is there).
#pragma once
#include "common.h"

namespace moba {

constexpr int kLeastPageLog2 = 4, kMostPageLog2 = 8;
constexpr float kE4m3Max = 448.f;
constexpr int kLeastScaleExponent = -100;

struct PageTable {
  const int32_t* pages;    // [B] rows of `stride` entries
  const int32_t* lengths;  // [B]
  const int32_t* cu_new;   // [B+1]
  int64_t stride;
  int B, T;                // sequences, packed rows
  int num_pages, max_pages, page_log2;
};

// rows lo .. hi - 1 are the sequence's new tokens; token t of them is its position length - hi + t
struct Sequence {
  int lo, hi;
  int64_t length;
};
__device__ __forceinline__ Sequence sequence_of(const PageTable& t, int b) {
  Sequence s;
  s.lo = min(max(t.cu_new[b], 0), t.T);
  s.hi = min(max(t.cu_new[b + 1], s.lo), t.T);
  s.length = max(t.lengths[b], 0);
  return s;
}
// tokens that the sequence's row of the table has room for
__device__ __forceinline__ int64_t room(const PageTable& t) { return (int64_t)t.max_pages << t.page_log2; }
// id of a sequence's page, -1 where the table names none
__device__ __forceinline__ int page_id(const PageTable& t, int b, int64_t page) {
  if (page < 0 || page >= t.max_pages) return -1;
  const int id = t.pages[b * t.stride + page];
  return id >= 0 && id < t.num_pages ? id : -1;
}

// The last sequence b with start(b, cu_new[b]) <= x, for ascending starts, its row range and length, found by the lanes of a
// wave together with one round of loads for every 64 sequences; b = -1 if there is none.
template <class Start>
__device__ __forceinline__ int last_up_to(const PageTable& t, int64_t x, int lane, Sequence& seq, Start start) {
  int found = -1;
  for (int b0 = 0; b0 < t.B; b0 += 64) {
    const int b = min(b0 + lane, t.B - 1);
    const Sequence s = sequence_of(t, b);
    const uint64_t m = __ballot(b0 + lane < t.B && start(b, s.lo) <= x);
    if (m) {
      const int at = 63 - __builtin_clzll(m);
      found = b0 + at;
      seq.lo = __builtin_amdgcn_readlane(s.lo, at);
      seq.hi = __builtin_amdgcn_readlane(s.hi, at);
      seq.length = __builtin_amdgcn_readlane((int)s.length, at);
    }
    if (~m) break;
  }
  return found;
}

inline int page_log2_of(int page_size) {
  for (int l = kLeastPageLog2; l <= kMostPageLog2; ++l)
    if (page_size == 1 << l) return l;
  return -1;
}

}  // namespace moba
