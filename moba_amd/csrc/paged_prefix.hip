// Attention of new tokens over the paged cache where sequences begin with the same pages: what they share is read once for all of
// them, by the kernels of paged_attn.h over the batch as paged_shared.h cuts it.  Sixteen users' tokens, 32 heads on 8, 8 bits, behind
// 32768 shared tokens and up to 8000 of their own: 133 MB in 39 us, of which the shared keys pass twice (64 rows of a key/value head,
// 32 to a workgroup), and the merge in 6.2; 33 us of the 39 are as many steps as the longest run has.  898 tokens of prompts behind
// 12288 and 69 of other users: products, 185 Gflop, 225 us (219 to 255 by the box), 24.6 for the few rows, 15.6 for the merge.
#include "paged_attn.h"
#include "paged_shared.h"

namespace moba {

// A token's rows with its group's keys, and with its sequence's.  Up to 64 sequences and groups are asked for at once.
__device__ __forceinline__ void sides_of(const Shape<SharedTable>& shape, int t, int lane, Side (&side)[2]) {
  const SharedTable& table = shape.table;
  Sequence seq = {}, all = {};
  int b = -1, g = -1;
  if (table.B <= 64 && table.G <= 64) {
    const Sequence mine = sequence_of(static_cast<const PageTable&>(table), min(lane, table.B - 1));
    const int group = min(lane, table.G - 1), first = table.cu_groups[group], end = table.cu_groups[group + 1];
    const int keys = shared_keys(table, group);
    const uint64_t begun = __ballot(lane < table.B && mine.lo <= t);
    if (begun) {
      b = 63 - __builtin_clzll(begun);
      seq = {__builtin_amdgcn_readlane(mine.lo, b), __builtin_amdgcn_readlane(mine.hi, b), __builtin_amdgcn_readlane((int)mine.length, b), 0};
      const uint64_t in = __ballot(lane < table.G && first <= b && b < end);
      if (in) {
        g = __ffsll((unsigned long long)in) - 1;
        const int m0 = min(max(__builtin_amdgcn_readlane(first, g), 0), table.B), m1 = max(min(__builtin_amdgcn_readlane(end, g), table.B), m0);
        all.lo = __builtin_amdgcn_readlane(mine.lo, min(m0, table.B - 1));     // (b is one of m0 .. m1 - 1)
        all.hi = __builtin_amdgcn_readlane(mine.hi, max(m1 - 1, 0));
        all.length = __builtin_amdgcn_readlane(keys, g);
      }
    }
  } else {
    b = last_up_to(table, t, lane, seq, [](int, int lo) { return (int64_t)lo; });
    g = b >= 0 ? __builtin_amdgcn_readfirstlane(group_of(table, b)) : -1;
    if (g >= 0) all = sequence_of(table, g);
  }
  const bool there = b >= 0 && t < seq.hi;
  const int keys = (int)min(seq.length, room(table)), begin = g >= 0 ? min((int)all.length, keys) : 0;
  side[0] = {max(g, 0), t - all.lo, all.hi - all.lo, there && g >= 0 && all.length > 0 && t >= all.lo && t < all.hi};
  side[1] = {table.G + max(b, 0), t - seq.lo, seq.hi - seq.lo, there && keys > begin};
}

// Units of the batch: its tokens are rows of a group and of a sequence.  Every unit leaves parts.
static Cuts shared_cuts(int64_t T, int B, int G, int rep, int Hkv, int D, bool cache8) {
  // More rows are few than where nothing is shared: the groups of 32 read the same keys at the same time, from L2 all but one.  Single tokens
  // of 24 sequences (96 rows) behind 16384 shared ones, 8 heads, 8 bits: 33 us as few rows, 49 as many; of 40 41 and 62, of 64 51 and
  // 70, of 128 87 and 103, but two pieces of 128 tokens 88 and 83.  16-bit elements, heads of 128: 40 sequences 55 and 71, 64 76 and 82,
  // but two pieces of 64 tokens 81 and 57.  Heads of 64: 64 rows to a workgroup (72 of four sequences behind 8208, fp16: 17.5 us with the
  // others' launch gone, 22.4 as many; heads of 128 have no registers for it: 66 us for 64 rows behind 32768, 39.8 in two groups).
  const int sets = few_sets<SharedTable>(D), few_rows = (D == 128 && !cache8 ? 4 : 8) * kFewRows;
  Cuts c = paged_cuts(2 * T, B + G, rep, Hkv, D, cache8, T * rep > few_rows, sets * kFewRows, few_rows, D == 128 && !cache8 ? 1 : 2);
  if (c.many.most > 0) {   // (pieces of prompts behind what is shared, among others: units of many lengths)
    c.many.even = true;
    const int64_t most = c.many.most + 2 * (int64_t)c.many.target;
    c.many.most = (int)(most < 0x7fffffff ? most : 0x7fffffff);
  }
  c.few.parts = c.few.most;
  c.many.parts = c.many.most;
  return c;
}
static bool sizes_ok(int64_t T, int B, int G, int H, int Hkv) {
  return paged_sizes_ok(T, B, H, Hkv) && G > 0;
}

template <class E>
static int prefix_attention(PagedParams<E, SharedTable>& p, const void* q, void* out, const void* k_pages, const void* v_pages,
                            const float* k_scales, const float* v_scales, char* workspace, int D, const int64_t* strides, int cache8,
                            float scale, hipStream_t st) {
  const SharedTable& table = p.shape.table;
  const Cuts cuts = shared_cuts(table.T, table.B, table.G, p.shape.rep, p.shape.Hkv, D, cache8 != 0);
  if (!set_params(p, cuts, q, out, k_pages, v_pages, k_scales, v_scales, workspace, table.B + table.G, D, strides, cache8 != 0, scale))
    return MOBA_ERR_LIMIT;
  if (D == 128) return cache8 ? launch_paged<E, 128, true>(p, st) : launch_paged<E, 128, false>(p, st);
  return cache8 ? launch_paged<E, 64, true>(p, st) : launch_paged<E, 64, false>(p, st);
}

}  // namespace moba

using namespace moba;

extern "C" size_t moba_paged_prefix_attention_workspace_bytes(int64_t T, int B, int G, int H, int Hkv, int D, int cache8) {
  if (!sizes_ok(T, B, G, H, Hkv) || (D != 64 && D != 128) || T >= 1 << 24 || (int64_t)B + G >= 1LL << 31) return 0;
  return paged_workspace_bytes(shared_cuts(T, B, G, H / Hkv, Hkv, D, cache8 != 0), B + G, Hkv, D);
}

// strides, in elements: {q token, q head, page table row}
extern "C" int moba_paged_prefix_attention(const void* q, void* out, const void* k_pages, const void* v_pages, const float* k_scales,
                                           const float* v_scales, const int32_t* page_table, const int32_t* lengths,
                                           const int32_t* cu_new, const int32_t* cu_groups, const int32_t* shared, void* workspace,
                                           int64_t T, int B, int G, int H, int Hkv, int D, int page_size, int64_t num_pages,
                                           int64_t max_pages, const int64_t* strides, int cache8, float scale, int dtype, void* stream) {
  if (!cu_groups || !shared || G <= 0) return MOBA_ERR_ARG;
  PageTable table;
  const int rc = check_paged(table, q, out, k_pages, v_pages, k_scales, v_scales, page_table, lengths, cu_new, workspace, T, B, H, Hkv, D,
                             page_size, num_pages, max_pages, strides, cache8, dtype);
  if (rc != MOBA_OK) return rc;
  if ((int64_t)B + G >= 1LL << 31) return MOBA_ERR_LIMIT;
  const SharedTable both = {table, cu_groups, shared, G};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MOBA_DTYPE_F16) {
    PagedParams<F16, SharedTable> p = {};
    p.shape = {both, H, Hkv, H / Hkv};
    return prefix_attention(p, q, out, k_pages, v_pages, k_scales, v_scales, (char*)workspace, D, strides, cache8, scale, st);
  }
  PagedParams<Bf16, SharedTable> p = {};
  p.shape = {both, H, Hkv, H / Hkv};
  return prefix_attention(p, q, out, k_pages, v_pages, k_scales, v_scales, (char*)workspace, D, strides, cache8, scale, st);
}
