// Attention of new tokens over the paged cache where sequences begin with the same pages: what they share is read once for all of
// them, by the kernels of paged_attn.h over the batch as paged_shared.h cuts it.
#include "paged_attn.h"
#include "paged_shared.h"

namespace moba {

// a token's rows with its group's keys, and with its sequence's
__device__ __forceinline__ void sides_of(const Shape<SharedTable>& shape, int t, int lane, Side (&side)[2]) {
  const SharedTable& table = shape.table;
  Sequence seq = {};
  const int b = last_up_to(table, t, lane, seq, [](int, int lo) { return (int64_t)lo; });
  const bool there = b >= 0 && t < seq.hi;
  const int g = there ? __builtin_amdgcn_readfirstlane(group_of(table, b)) : -1;
  side[0] = side[1] = {0, 0, 0, false};
  int begin = 0;
  const int keys = (int)min(seq.length, room(table));
  if (g >= 0) {
    const Sequence all = sequence_of(table, g);
    side[0] = {g, t - all.lo, all.hi - all.lo, all.length > 0 && t >= all.lo && t < all.hi};
    begin = min((int)all.length, keys);
  }
  if (there) side[1] = {table.G + b, t - seq.lo, seq.hi - seq.lo, keys > begin};
}

// Units of the batch: its tokens are rows of a group and of a sequence.  Every unit leaves parts.
static Cuts shared_cuts(int64_t T, int B, int G, int rep, int Hkv, int D, bool cache8) {
  Cuts c = paged_cuts(2 * T, B + G, rep, Hkv, D, cache8, -1);
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
