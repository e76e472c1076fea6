// Attention of new tokens over the blocks of the paged cache that each of their rows has chosen (the reference attends such blocks
// of whole prompts: moba/moba_efficient.py:373-443): the few-row kernel of paged_attn.h over lists of blocks (paged_chosen.h).  Bound by
// memory as the attention over all keys is, on fewer bytes.
#include "paged_attn.h"
#include "paged_chosen.h"

namespace moba {

constexpr int kMostTopk = 64;
constexpr int64_t kListsAtOnce = 1LL << 29;   // bytes of a launch's lists in memory: more units are several launches
static_assert(64 * kFewWaves == kListThreads && kLdsEntries * sizeof(Chosen) == kListBytes);
static_assert(few_list_at<64, true>() >= 4 * kWindow + 64);

// Sizes that follow from a batch's bounds
struct ChosenSizes {
  Cuts cuts;
  int room_of_list;     // 0: in LDS
  int units;            // of a launch
  int64_t lists_at, bytes;
};
static ChosenSizes chosen_sizes(int64_t T, int B, int rep, int Hkv, int D, int64_t max_pages, int each, int topk, bool cache8) {
  ChosenSizes s;
  s.cuts = paged_cuts(T, B, rep, Hkv, D, cache8, false, kChosenRows, 0, D == 128 && !cache8 ? 1 : 2);
  const int64_t rows = T * rep < kChosenRows ? T * rep : kChosenRows, blocks = (max_pages - 1) / each + 1;
  const int64_t room = rows * topk < blocks ? rows * topk : blocks;
  s.room_of_list = room > kLdsEntries ? (int)room : 0;
  s.lists_at = ((int64_t)paged_workspace_bytes(s.cuts, B, Hkv, D) + 15) / 16 * 16;
  const int64_t list = s.room_of_list * (int64_t)sizeof(Chosen);
  int64_t units = ((1 << 24) - 1) / Hkv;   // (2^32 threads)
  if (list && units > kListsAtOnce / (list * Hkv)) units = std::max(kListsAtOnce / (list * Hkv), (int64_t)1);
  s.units = (int)std::min(units, (int64_t)s.cuts.few.most);
  s.bytes = s.lists_at + s.units * Hkv * list;
  return s;
}

template <class E>
static int block_attention(const ChosenTable& table, const ChosenSizes& s, const void* q, void* out, const void* k_pages,
                           const void* v_pages, const float* k_scales, const float* v_scales, char* workspace, int H, int Hkv, int D,
                           const int64_t* strides, int cache8, float scale, hipStream_t st) {
  PagedParams<E, ChosenTable> p = {};
  p.shape = {table, H, Hkv, H / Hkv};
  if (!set_params(p, s.cuts, q, out, k_pages, v_pages, k_scales, v_scales, workspace, table.B, D, strides, cache8 != 0, scale))
    return MOBA_ERR_LIMIT;
  if (D == 128) return cache8 ? launch_paged<E, 128, true>(p, st) : launch_paged<E, 128, false>(p, st);
  return cache8 ? launch_paged<E, 64, true>(p, st) : launch_paged<E, 64, false>(p, st);
}

static int check_blocks(int64_t T, int B, int H, int Hkv, int page_size, int64_t max_pages, int block_size, int topk) {
  if (!paged_sizes_ok(T, B, H, Hkv) || max_pages <= 0 || topk <= 0) return MOBA_ERR_ARG;
  if (page_log2_of(page_size) < 0 || block_size <= 0 || block_size % page_size) return MOBA_ERR_UNSUPPORTED;
  if (T >= 1LL << 24 || T * H >= 1LL << 31 || max_pages >= 1LL << 31 || topk > kMostTopk || block_size > 1 << 24 ||
      (int64_t)B * Hkv >= 1LL << 24)
    return MOBA_ERR_LIMIT;
  return MOBA_OK;
}

}  // namespace moba

using namespace moba;

extern "C" size_t moba_paged_block_attention_workspace_bytes(int64_t T, int B, int H, int Hkv, int D, int page_size, int64_t max_pages,
                                                             int block_size, int topk, int cache8) {
  if (check_blocks(T, B, H, Hkv, page_size, max_pages, block_size, topk) != MOBA_OK || (D != 64 && D != 128)) return 0;
  return (size_t)chosen_sizes(T, B, H / Hkv, Hkv, D, max_pages, block_size / page_size, topk, cache8 != 0).bytes;
}

// strides, in elements: {q token, q head, page table row}
extern "C" int moba_paged_block_attention(const void* q, void* out, const void* k_pages, const void* v_pages, const float* k_scales,
                                          const float* v_scales, const int32_t* blocks, const int32_t* page_table,
                                          const int32_t* lengths, const int32_t* cu_new, void* workspace, int64_t T, int B, int H, int Hkv,
                                          int D, int page_size, int64_t num_pages, int64_t max_pages, int block_size, int topk,
                                          const int64_t* strides, int cache8, float scale, int dtype, void* stream) {
  if (!blocks) return MOBA_ERR_ARG;
  PageTable table;
  int rc = check_paged(table, q, out, k_pages, v_pages, k_scales, v_scales, page_table, lengths, cu_new, workspace, T, B, H, Hkv, D, page_size,
                       num_pages, max_pages, strides, cache8, dtype);
  if (rc == MOBA_OK) rc = check_blocks(T, B, H, Hkv, page_size, max_pages, block_size, topk);
  if (rc != MOBA_OK) return rc;
  const int each = block_size / page_size;
  const ChosenSizes s = chosen_sizes(T, B, H / Hkv, Hkv, D, max_pages, each, topk, cache8 != 0);
  char* const space = (char*)workspace;
  const ChosenTable chosen = {table, blocks, s.room_of_list ? (Chosen*)(space + s.lists_at) : nullptr, topk, each, divisor_or_one(each),
                              s.room_of_list, 0, s.units};
  hipStream_t st = (hipStream_t)stream;
  return dtype == MOBA_DTYPE_F16
             ? block_attention<F16>(chosen, s, q, out, k_pages, v_pages, k_scales, v_scales, space, H, Hkv, D, strides, cache8, scale, st)
             : block_attention<Bf16>(chosen, s, q, out, k_pages, v_pages, k_scales, v_scales, space, H, Hkv, D, strides, cache8, scale, st);
}
