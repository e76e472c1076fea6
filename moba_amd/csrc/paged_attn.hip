// Entry points of the attention over the paged cache (paged_attn.h).
#include "paged_attn.h"

namespace moba {

static Cuts whole_cuts(int64_t T, int B, int rep, int Hkv, int D, bool cache8, int max_new) {
  const int64_t most_new = max_new >= 0 && max_new < T ? max_new : T;
  // 8-bit pages: up to 64 rows are few, in two groups of which the second finds the keys in L2.  16 sequences of 64 rows against 8192
  // keys, 8 heads: 100 us, as many rows 112; 64 of 40 against 2048: 86 and 101; one of 64 against 131072, one head: 30 and 32.  128
  // rows would be faster for 8 heads (one sequence, 4096 keys: 21 and 27) and slower for one (16 sequences, 8192 keys: 42 and 33).
  // 16-bit pages are twice the bytes: up to 32 rows (16 of 64 rows, one head: 30 us as many rows, 35 as few; 64 of 40: 110 and 135).
  const int few_rows = cache8 ? 2 * kFewRows : kFewRows;
  return paged_cuts(T, B, rep, Hkv, D, cache8, most_new * rep > few_rows, kFewRows, few_rows, D == 128 && !cache8 ? 1 : 2);
}

}  // namespace moba

using namespace moba;

extern "C" size_t moba_paged_attention_workspace_bytes(int64_t T, int B, int H, int Hkv, int D, int cache8, int max_new) {
  if (!paged_sizes_ok(T, B, H, Hkv) || (D != 64 && D != 128)) return 0;
  const Cuts c = whole_cuts(T, B, H / Hkv, Hkv, D, cache8 != 0, max_new);
  return paged_workspace_bytes(c, B, Hkv, D);
}

template <class E>
static int paged_attention(const void* q, void* out, const void* k_pages, const void* v_pages, const float* k_scales,
                           const float* v_scales, const PageTable& table, char* workspace, int H, int Hkv, int D, int max_new,
                           const int64_t* strides, int cache8, float scale, hipStream_t st) {
  PagedParams<E> p = {};
  p.shape = {table, H, Hkv, H / Hkv};
  const Cuts cuts = whole_cuts(table.T, table.B, p.shape.rep, Hkv, D, cache8 != 0, max_new);
  if (!set_params(p, cuts, q, out, k_pages, v_pages, k_scales, v_scales, workspace, table.B, D, strides, cache8 != 0, scale))
    return MOBA_ERR_LIMIT;
  if (D == 128) return cache8 ? launch_paged<E, 128, true>(p, st) : launch_paged<E, 128, false>(p, st);
  return cache8 ? launch_paged<E, 64, true>(p, st) : launch_paged<E, 64, false>(p, st);
}

// strides, in elements: {q token, q head, page table row}
extern "C" int moba_paged_attention(const void* q, void* out, const void* k_pages, const void* v_pages, const float* k_scales,
                                    const float* v_scales, const int32_t* page_table, const int32_t* lengths,
                                    const int32_t* cu_new, void* workspace, int64_t T, int B, int H, int Hkv, int D, int page_size,
                                    int64_t num_pages, int64_t max_pages, int max_new, const int64_t* strides, int cache8,
                                    float scale, int dtype, void* stream) {
  PageTable table;
  const int rc = check_paged(table, q, out, k_pages, v_pages, k_scales, v_scales, page_table, lengths, cu_new, workspace, T, B, H, Hkv, D,
                             page_size, num_pages, max_pages, strides, cache8, dtype);
  if (rc != MOBA_OK) return rc;
  hipStream_t st = (hipStream_t)stream;
  return dtype == MOBA_DTYPE_F16
             ? paged_attention<F16>(q, out, k_pages, v_pages, k_scales, v_scales, table, (char*)workspace, H, Hkv, D, max_new,
                                    strides, cache8, scale, st)
             : paged_attention<Bf16>(q, out, k_pages, v_pages, k_scales, v_scales, table, (char*)workspace, H, Hkv, D, max_new,
                                     strides, cache8, scale, st);
}
