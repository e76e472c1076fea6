// Attention of new tokens over the blocks of the paged cache that each of their rows has chosen (the reference attends such blocks
// of whole prompts: moba/moba_efficient.py:373-443).
//
// The union of up to 32 rows' blocks becomes a list (paged_union_kernel): a mask of rows for every block of the sequence, in LDS, a
// window at a time, into which the rows' entries are or-ed (whatever their order, one result), and of which the blocks with a
// row are counted through.  Then the few-row kernel of paged_attn.h reads the list's keys once, every row masked to what it has
// chosen, and the merge puts the runs together.  Bound by memory as the attention over all keys is, on fewer bytes.
#include "paged_attn.h"
#include "paged_chosen.h"

namespace moba {

constexpr int kUnionThreads = 256, kWindow = 4096;   // blocks of a window
constexpr int kMostTopk = 64;

struct UnionParams {
  Shape<ChosenTable> shape;
  Chosen* lists;
  int32_t* keys;
  Runs* runs;
};

__global__ __launch_bounds__(kUnionThreads) void paged_union_kernel(const UnionParams p) {
  constexpr int kEach = kWindow / kUnionThreads;
  __shared__ uint32_t mask[kWindow];
  __shared__ int sums[kUnionThreads / 64];
  __shared__ int last_block;
  const auto& shape = p.shape;
  const ChosenTable& t = shape.table;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int g = blockIdx.x, hkv = blockIdx.y, item = g * shape.Hkv + hkv;
  Sequence seq = {};
  const int b = last_up_to(t, g, lane, seq, [&](int at, int lo) { return first_group(lo, shape.rep, at); });
  const int64_t row0 = b < 0 ? 0 : (g - first_group(seq.lo, shape.rep, b)) * kChosenRows;
  const int64_t count = b < 0 ? 0 : (int64_t)(seq.hi - seq.lo) * shape.rep;
  const int rows_here = (int)min(max(count - row0, (int64_t)0), (int64_t)kChosenRows);
  const int keys = rows_here ? keys_of(shape, seq) : 0, block_keys = t.each << t.page_log2;
  const int blocks = keys > 0 ? (keys - 1) / block_keys + 1 : 0;
  int total = 0;
  for (int w0 = 0; w0 < blocks; w0 += kWindow) {
    const int here = min(kWindow, blocks - w0);
    for (int i = tid; i < (here + kEach - 1) / kEach * kEach; i += kUnionThreads) mask[i] = 0;
    __syncthreads();
    for (int i = tid; i < rows_here * t.K; i += kUnionThreads) {
      const int r = i / t.K, row = (int)row0 + r, j = row / shape.rep;
      const int64_t position = seq.length - (seq.hi - seq.lo) + j;
      const int block = t.blocks[((int64_t)(seq.lo + j) * shape.H + hkv * shape.rep + row - j * shape.rep) * t.K + i - r * t.K];
      if (block >= w0 && block < w0 + here && (int64_t)block * block_keys <= position) atomicOr(&mask[block - w0], 1u << r);
    }
    __syncthreads();
    // each thread its neighbouring blocks
    int mine = 0;
    if (tid * kEach < here)
#pragma unroll
      for (int k = 0; k < kEach; ++k) mine += mask[tid * kEach + k] != 0;
    int upto = (int)upto_sum(mine);
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < kUnionThreads / 64; ++w) {
      if (w < wave) upto += sums[w];
      all += sums[w];
    }
    int at = total + upto - mine;
    if (tid * kEach < here)
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        const uint32_t who = mask[tid * kEach + k];
        if (!who) continue;
        p.lists[(int64_t)item * t.room_of_list + at] = {w0 + tid * kEach + k, who};
        if (++at == total + all) last_block = w0 + tid * kEach + k;
      }
    total += all;
    __syncthreads();   // (the masks and sums have been read)
  }
  if (tid == 0) {
    p.keys[item] = total ? (total - 1) * block_keys + min(block_keys, keys - last_block * block_keys) : 0;
    p.runs[item] = {0, 0, 0};
  }
}

// a row's parts by its group and key/value head
template <class E>
struct MergeToken<E, ChosenTable> {
  Sequence seq;
  int b, token;
  __device__ __forceinline__ MergeToken(const PagedParams<E, ChosenTable>& p, int t, int lane) {
    seq = {};
    b = last_up_to(p.shape.table, t, lane, seq, [](int, int lo) { return (int64_t)lo; });
    if (t >= seq.hi) b = -1;
    token = t - seq.lo;
  }
  __device__ __forceinline__ bool done() const { return false; }
  __device__ __forceinline__ Parts parts(const PagedParams<E, ChosenTable>& p, int hkv, int g, int) const {
    const Shape<ChosenTable>& shape = p.shape;
    Runs r = {0, 0, 0};
    const int row = token * shape.rep + g, group = row / kChosenRows;
    if (b >= 0) {
      const int64_t item = (first_group(seq.lo, shape.rep, b) + group) * shape.Hkv + hkv;
      if (item < shape.table.items) r = p.runs[item];
    }
    if (r.runs > 1 && (int64_t)r.first + r.runs > p.few.parts) r.runs = 0;   // (cannot be)
    return {p.few_o, p.few_lse, r.runs, (int64_t)r.first * kChosenRows + row - group * kChosenRows, kChosenRows};
  }
};

// Sizes that follow from a batch's bounds
struct ChosenSizes {
  int items, room_of_list;
  Cut cut;
  int64_t lists_at, keys_at, parts_at, bytes;   // the runs lie first
};
static bool chosen_sizes(ChosenSizes& s, int64_t T, int B, int H, int Hkv, int D, int page_size, int64_t max_pages, int block_size, int topk,
                         bool cache8) {
  const int64_t items = (T * (H / Hkv) / kChosenRows + B) * Hkv, blocks = (max_pages - 1) / (block_size / page_size) + 1;
  const int64_t room = (int64_t)kChosenRows * topk < blocks ? (int64_t)kChosenRows * topk : blocks;
  const int cus = compute_units() > 0 ? compute_units() : 256, target = (D == 128 && !cache8 ? 1 : 2) * cus;
  if (items >= 1LL << 24) return false;   // (2^32 threads)
  s.items = (int)items;
  s.room_of_list = (int)room;
  const int64_t most = items >= (int64_t)kWholeAt * target ? items : target / 2 + items > target ? target / 2 + items : target;
  s.cut = {kChosenRows, kFewTile, 2, 0, 0x7fffffff, target, (int)most, items >= (int64_t)kWholeAt * target ? 0 : (int)most, false};
  auto lines = [](int64_t n) { return (n + 15) / 16 * 16; };
  s.lists_at = lines(items * (int64_t)sizeof(Runs));
  s.keys_at = s.lists_at + lines(items * room * (int64_t)sizeof(Chosen));
  s.parts_at = s.keys_at + lines(items * 4);
  s.bytes = s.parts_at + (int64_t)s.cut.parts * kChosenRows * (D + 1) * 4;
  return true;
}

template <class E, int D, bool k8>
static int launch_chosen(const PagedParams<E, ChosenTable>& p, const UnionParams& u, hipStream_t st) {
  LaunchCheck launch_check;
  static bool allowed[kMaxDevices];
  const auto few = paged_few_kernel<E, D, k8, ChosenTable, 1>;
  if (!allow_dynamic_lds((const void*)few, few_lds_bytes<D, k8>(), allowed)) return MOBA_ERR_LAUNCH;
  hipLaunchKernelGGL(paged_union_kernel, dim3(p.shape.table.items / p.shape.Hkv, p.shape.Hkv), dim3(kUnionThreads), 0, st, u);
  hipLaunchKernelGGL(few, dim3((unsigned)p.few.most), dim3(64 * kFewWaves), (few_lds_bytes<D, k8>()), st, p);
  launch_merge<E, D>(p, st);
  return launch_check.result();
}

template <class E>
static int block_attention(const ChosenTable& table, const ChosenSizes& s, const void* q, void* out, const void* k_pages,
                           const void* v_pages, const float* k_scales, const float* v_scales, char* workspace, int H, int Hkv, int D,
                           const int64_t* strides, int cache8, float scale, hipStream_t st) {
  typedef typename E::elem elem;
  PagedParams<E, ChosenTable> p = {};
  p.shape = {table, H, Hkv, H / Hkv};
  p.few = s.cut;
  p.q = (const elem*)q; p.out = (elem*)out;
  p.pages[0] = (const char*)k_pages; p.pages[1] = (const char*)v_pages;
  p.scales[0] = k_scales; p.scales[1] = v_scales;
  p.runs = (Runs*)workspace;
  p.few_o = (float*)(workspace + s.parts_at);
  p.few_lse = p.few_o + (int64_t)s.cut.parts * kChosenRows * D;
  p.q_tok_stride = strides[0]; p.q_head_stride = strides[1];
  p.scale_log2 = scale * 1.4426950408889634f;
  const UnionParams u = {p.shape, (Chosen*)(workspace + s.lists_at), (int32_t*)(workspace + s.keys_at), p.runs};
  if (D == 128) return cache8 ? launch_chosen<E, 128, true>(p, u, st) : launch_chosen<E, 128, false>(p, u, st);
  return cache8 ? launch_chosen<E, 64, true>(p, u, st) : launch_chosen<E, 64, false>(p, u, st);
}

static int check_blocks(int64_t T, int B, int H, int Hkv, int page_size, int64_t max_pages, int block_size, int topk) {
  if (!paged_sizes_ok(T, B, H, Hkv) || max_pages <= 0 || topk <= 0) return MOBA_ERR_ARG;
  if (page_log2_of(page_size) < 0 || block_size <= 0 || block_size % page_size) return MOBA_ERR_UNSUPPORTED;
  if (T >= 1LL << 24 || T * H >= 1LL << 31 || max_pages >= 1LL << 31 || topk > kMostTopk || block_size > 1 << 24 || Hkv > 65535)
    return MOBA_ERR_LIMIT;
  return MOBA_OK;
}

}  // namespace moba

using namespace moba;

extern "C" size_t moba_paged_block_attention_workspace_bytes(int64_t T, int B, int H, int Hkv, int D, int page_size, int64_t max_pages,
                                                             int block_size, int topk, int cache8) {
  ChosenSizes s;
  if (check_blocks(T, B, H, Hkv, page_size, max_pages, block_size, topk) != MOBA_OK || (D != 64 && D != 128) ||
      !chosen_sizes(s, T, B, H, Hkv, D, page_size, max_pages, block_size, topk, cache8 != 0))
    return 0;
  return (size_t)s.bytes;
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
  ChosenSizes s;
  if (!chosen_sizes(s, T, B, H, Hkv, D, page_size, max_pages, block_size, topk, cache8 != 0)) return MOBA_ERR_LIMIT;
  char* const space = (char*)workspace;
  const int each = block_size / page_size;
  const ChosenTable chosen = {table, blocks, (const Chosen*)(space + s.lists_at), (const int32_t*)(space + s.keys_at), topk, each,
                              divisor_or_one(each), s.room_of_list, s.items, s.cut.target};
  hipStream_t st = (hipStream_t)stream;
  return dtype == MOBA_DTYPE_F16
             ? block_attention<F16>(chosen, s, q, out, k_pages, v_pages, k_scales, v_scales, space, H, Hkv, D, strides, cache8, scale, st)
             : block_attention<Bf16>(chosen, s, q, out, k_pages, v_pages, k_scales, v_scales, space, H, Hkv, D, strides, cache8, scale, st);
}
