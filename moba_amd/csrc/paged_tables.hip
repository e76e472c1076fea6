// Pages for new tokens from a pool, and back: the page table, the lengths, and where every new token belongs, from the sequences' lengths
// on the device.
//
// The pool is a stack of page numbers, free_pages [num_pages], of which the first free_count are free.  Reserve, with P tokens to a page:
//   n_b    = new_b, 0 where old_b + n_b tokens do not fit the sequence's row of the table (or 31 bits)
//   need_b = ceil((old_b + n_b) / P) - ceil(old_b / P)
//   b is served if sum_{i<=b} n_i <= rows and (need_b = 0 or sum_{i<=b} need_i <= free_count), and gets nothing otherwise
// Page number i that is given out (the served sequences' in order) is the i-th from the top.  Release is the inverse: the pages
// of a sequence behind its first `keep` tokens go back so that the first sequence's first page is on top again.
//
// One workgroup decides: the sums over the sequences are scans in registers (of 32 bits that saturate: what is compared with a limit
// may stop there) with one number of every wave in LDS.  For up to kRowsAtOnce rows it also fills the table and says where the rows
// belong; more are a second launch of as many workgroups as that takes, which finds ranks and rows in what the first has left.
// A row's page is looked up where it comes from, the table or the pool's stack, and waits for no entry to be written.  Nothing here
// is floating point, and no order depends on timing.  Bound by latency: 64 sequences with five tokens each 4.3 us, their way back 3.0
// (with 64-bit sums by lane shuffles, and rows that waited for the table, 10.4; entries that each look for their sequence, 4.1 back);
// eight documents of 471000 tokens on 29000 pages of 16 tokens 3.1 + 7.5 us, and 10.1 back (16.3), by one workgroup, as a page's place
// on the stack is the number of those before it; more entries of a thread on their way at once, 16, are 20.8, four 12.1.
#include "common.h"
#include "paged_cut.h"

namespace moba {

constexpr int kTableThreads = 1024, kTableWaves = kTableThreads / 64;
constexpr int kMostTableSequences = 8192;   // whose sums fit a workgroup's LDS
// (8000 rows 6.1 us, 3.0 + 4.4 with the second launch; 4000 4.8, 2.9 + 4.4)
constexpr int kRowsAtOnce = 8192;
constexpr int kPagesOfThread = 8;           // that a thread takes back at a time, where there are more than threads

struct Pool {
  int32_t* free_pages;   // [num_pages]
  int32_t* free_count;   // [1]
  int num_pages;
};
struct TableParams {
  Pool pool;
  int32_t* table;        // [B] rows of `stride` entries
  int32_t* lengths;      // [B]
  const int32_t* asked;  // [B]: new tokens, or those to keep
  int32_t *cu_new, *owners, *positions;   // [B+1], [rows], [rows]
  int64_t* slots;        // [rows]
  int32_t* ranks;        // [B+1]: number of the first page given to a sequence, and of all of them
  int64_t stride;
  int B, rows, max_pages, page_log2;
};

// Sums over the threads up to this one, and over all of them, of two numbers at a time
struct Two {
  uint32_t a, b;
};
struct Scan {
  Two upto, all;
};
__device__ __forceinline__ uint32_t add_sat(uint32_t x, uint32_t y) { return __builtin_elementwise_add_sat(x, y); }
// the lanes' sums as upto_sum() has them, saturating
__device__ __forceinline__ uint32_t upto_sat(uint32_t x) {
#define MOBA_DPP_ADD(ctrl, rows) x = add_sat(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, false))
  MOBA_DPP_ADD(0x111, 0xf);
  MOBA_DPP_ADD(0x112, 0xf);
  MOBA_DPP_ADD(0x114, 0xf);
  MOBA_DPP_ADD(0x118, 0xf);
  MOBA_DPP_ADD(0x142, 0xa);
  MOBA_DPP_ADD(0x143, 0xc);
#undef MOBA_DPP_ADD
  return x;
}
// red: [waves], another one than in the call before; every thread calls it
__device__ __forceinline__ Scan scan(Two x, Two* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  x = {upto_sat(x.a), upto_sat(x.b)};
  if (lane == 63) red[wave] = x;
  __syncthreads();
  Two before = {0, 0}, all = {0, 0};
#pragma unroll
  for (int w = 0; w < kTableWaves; ++w) {
    const Two y = red[w];
    before = {w < wave ? add_sat(before.a, y.a) : before.a, w < wave ? add_sat(before.b, y.b) : before.b};
    all = {add_sat(all.a, y.a), add_sat(all.b, y.b)};
  }
  return {{add_sat(x.a, before.a), add_sat(x.b, before.b)}, all};
}

// the last i in [0, n) with a[i] <= x, for ascending a with a[0] <= x
__device__ __forceinline__ int last_at_most(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(int64_t tokens, int page_log2) { return (int)((tokens + (1 << page_log2) - 1) >> page_log2); }

// Row t of a batch whose row ranges, given pages and former lengths are cu, rank [B+1] and old(b); top: free pages before the call
template <class Old>
__device__ __forceinline__ void place_row(const TableParams& p, const int* cu, const int* rank, Old old, int top, int t) {
  int b = -1, position = 0;
  int64_t slot = -1;
  if (t < cu[p.B]) {
    b = last_at_most(cu, p.B, t);
    const int before = old(b), have = pages_of(before, p.page_log2);
    position = before + t - cu[b];
    const int page = position >> p.page_log2;
    const int id = page < have ? p.table[b * p.stride + page] : p.pool.free_pages[top - 1 - (rank[b] + page - have)];
    if (id >= 0 && id < p.pool.num_pages) slot = ((int64_t)id << p.page_log2) + (position & ((1 << p.page_log2) - 1));
  }
  p.owners[t] = b;
  p.positions[t] = position;
  p.slots[t] = slot;
}
// Pages i .. of those that are given, up to `end`, go to their entries
template <class Old>
__device__ __forceinline__ void place_pages(const TableParams& p, const int* rank, Old old, int top, int i, int end) {
  if (i >= end) return;
  for (int b = last_at_most(rank, p.B, i); i < end; ++i) {
    while (rank[b + 1] <= i) ++b;   // (some sequence has page i: i < rank[B])
    p.table[b * p.stride + pages_of(old(b), p.page_log2) + i - rank[b]] = p.pool.free_pages[top - 1 - i];
  }
}

__global__ __launch_bounds__(kTableThreads) void paged_reserve_kernel(const TableParams p) {
  __shared__ Two red[2][kTableWaves];
  extern __shared__ int lds[];
  int* const cu = lds;                       // [B+1]
  int* const rank = cu + p.B + 1;            // [B+1]
  int* const old_length = rank + p.B + 1;    // [B]
  const int tid = threadIdx.x;
  const int top = min(max(*p.pool.free_count, 0), p.pool.num_pages);
  const int64_t most = min((int64_t)p.max_pages << p.page_log2, (int64_t)0x7fffffff);
  Two asked = {0, 0}, given = {0, 0};   // tokens and pages, of the sequences of the steps before
  for (int b0 = 0; b0 < p.B; b0 += kTableThreads) {
    const int b = b0 + tid;
    int64_t old = 0, n = 0;
    if (b < p.B) {
      old = max(p.lengths[b], 0);
      n = max(p.asked[b], 0);
      if (old + n > most) n = 0;
    }
    const uint32_t need = pages_of(old + n, p.page_log2) - pages_of(old, p.page_log2);
    const Scan wanted = scan({(uint32_t)n, need}, red[0]);
    const bool served = add_sat(asked.a, wanted.upto.a) <= (uint32_t)p.rows &&
                        (need == 0 || add_sat(asked.b, wanted.upto.b) <= (uint32_t)top);
    asked = {add_sat(asked.a, wanted.all.a), add_sat(asked.b, wanted.all.b)};
    const Scan got = scan({served ? (uint32_t)n : 0, served ? need : 0}, red[1]);   // (below 2^31)
    if (b < p.B) {
      const int end = (int)(given.a + got.upto.a), pages = (int)(given.b + got.upto.b);
      cu[b + 1] = end;
      rank[b + 1] = pages;
      old_length[b] = (int)old;
      p.cu_new[b + 1] = end;
      if (p.rows > kRowsAtOnce) p.ranks[b + 1] = pages;
      if (served && n) p.lengths[b] = (int)(old + n);
    }
    given = {given.a + got.all.a, given.b + got.all.b};
  }
  if (tid == 0) {
    cu[0] = rank[0] = p.cu_new[0] = 0;
    if (p.rows > kRowsAtOnce) p.ranks[0] = 0;
    *p.pool.free_count = top - (int)given.b;
  }
  if (p.rows > kRowsAtOnce) return;
  __syncthreads();
  auto old = [&](int b) { return old_length[b]; };
  for (int t = tid; t < p.rows; t += kTableThreads) place_row(p, cu, rank, old, top, t);
  for (int i = tid; i < (int)given.b; i += kTableThreads) place_pages(p, rank, old, top, i, i + 1);
}

// the same for rows, and pages, that are many: each thread four of them (there are no more pages than rows)
__global__ __launch_bounds__(256) void paged_rows_kernel(const TableParams p) {
  extern __shared__ int lds[];
  int *const cu = lds, *const rank = cu + p.B + 1, *const length = rank + p.B + 1;
  const int left = *p.pool.free_count;
  for (int b = threadIdx.x; b <= p.B; b += 256) {
    cu[b] = p.cu_new[b];
    rank[b] = p.ranks[b];
    if (b < p.B) length[b] = max(p.lengths[b], 0);
  }
  __syncthreads();
  const int top = left + rank[p.B];
  auto old = [&](int b) { return length[b] - (cu[b + 1] - cu[b]); };
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t t = (int64_t)blockIdx.x * 1024 + k * 256 + threadIdx.x;
    if (t < p.rows) place_row(p, cu, rank, old, top, (int)t);
  }
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i < rank[p.B]) place_pages(p, rank, old, top, (int)i, (int)min(i + 4, (int64_t)rank[p.B]));
}

__global__ __launch_bounds__(kTableThreads) void paged_release_kernel(const TableParams p) {
  __shared__ Two red[2][kTableWaves];
  __shared__ int counts[2][kTableWaves];
  extern __shared__ int lds[];
  int* const first = lds;                    // [B]: entries that go in the sequences before (their number is below 2^31)
  int* const stay = first + p.B;             // [B]: pages that stay
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int free_count = min(max(*p.pool.free_count, 0), p.pool.num_pages), total = 0, parity = 0;
  for (int b0 = 0; b0 < p.B; b0 += kTableThreads, parity ^= 1) {
    const int b = b0 + tid;
    int gone = 0, kept = 0;
    if (b < p.B) {
      const int old = max(p.lengths[b], 0), keep = min(max(p.asked[b], 0), old);
      kept = min(pages_of(keep, p.page_log2), p.max_pages);
      gone = min(pages_of(old, p.page_log2), p.max_pages) - kept;
      if (keep < old) p.lengths[b] = keep;
    }
    const Scan s = scan({(uint32_t)gone, 0}, red[parity]);
    if (b < p.B) {
      first[b] = total + (int)s.upto.a - gone;
      stay[b] = kept;
    }
    total += (int)s.all.a;
  }
  __syncthreads();
  // From the last entry to the first, so that a place on the stack is the number of pages that have come before.  A wave has neighbouring
  // entries, up to kPagesOfThread times its lanes of a step, and seldom has to look for their sequence.  (One compute unit's instructions are
  // what bounds it.)
  const int each = min((total + kTableThreads - 1) / kTableThreads, kPagesOfThread);
  int begin = 0, end = 0;          // entries of the sequence at hand
  int32_t* entries = nullptr;      // where entry 0 would be if all were its
  for (int64_t r0 = 0; r0 < total; r0 += kTableThreads * each, parity ^= 1) {
    int id[kPagesOfThread], found = 0;
    uint64_t valid[kPagesOfThread];
    const int last = (int)max(total - 1 - r0 - wave * each * 64 - lane, (int64_t)-1);
#pragma unroll
    for (int k = 0; k < kPagesOfThread; ++k) {
      if (k >= each) break;
      const int i = last - k * 64;
      id[k] = -1;
      if (i >= 0) {
        if (i < begin || i >= end) {
          const int b = last_at_most(first, p.B, i);
          begin = first[b];
          end = b + 1 < p.B ? first[b + 1] : total;
          entries = p.table + (b * p.stride + stay[b] - begin);
        }
        id[k] = entries[i];
        entries[i] = -1;
      }
    }
#pragma unroll
    for (int k = 0; k < kPagesOfThread; ++k) {
      if (k >= each) break;
      valid[k] = __ballot((uint32_t)id[k] < (uint32_t)p.pool.num_pages);
      found += __builtin_popcountll(valid[k]);
    }
    if (lane == 0) counts[parity][wave] = found;
    __syncthreads();
    const int mine = lane < kTableWaves ? counts[parity][lane] : 0, upto = (int)upto_sum((uint32_t)mine);
    int64_t place = (int64_t)free_count + __builtin_amdgcn_readlane(upto - mine, wave);
#pragma unroll
    for (int k = 0; k < kPagesOfThread; ++k) {
      if (k >= each) break;
      const int64_t to = place + __builtin_popcountll(valid[k] & ((1ull << lane) - 1));
      if ((valid[k] >> lane & 1) && to < p.pool.num_pages) p.pool.free_pages[to] = id[k];   // (more than there are: named twice)
      place += __builtin_popcountll(valid[k]);
    }
    free_count = (int)min((int64_t)free_count + __builtin_amdgcn_readlane(upto, 63), (int64_t)p.pool.num_pages);
  }
  if (tid == 0) *p.pool.free_count = free_count;
}

static int check_tables(TableParams& p, int32_t* free_pages, int32_t* free_count, int32_t* page_table, int32_t* lengths,
                        const int32_t* asked, int B, int page_size, int64_t num_pages, int64_t max_pages, int64_t table_stride) {
  if (!free_pages || !free_count || !page_table || !lengths || !asked || B <= 0 || num_pages <= 0 || max_pages <= 0 || table_stride < 0)
    return MOBA_ERR_ARG;
  const int page_log2 = page_log2_of(page_size);
  if (page_log2 < 0) return MOBA_ERR_UNSUPPORTED;
  if (B > kMostTableSequences || num_pages >= 1LL << 31 || max_pages >= 1LL << 31 || max_pages * B >= 1LL << 31) return MOBA_ERR_LIMIT;
  p = {};
  p.pool = {free_pages, free_count, (int)num_pages};
  p.table = page_table; p.lengths = lengths; p.asked = asked;
  p.stride = table_stride;
  p.B = B; p.max_pages = (int)max_pages; p.page_log2 = page_log2;
  return MOBA_OK;
}

}  // namespace moba

using namespace moba;

extern "C" size_t moba_paged_reserve_workspace_bytes(int B, int64_t rows) {
  return B > 0 && rows > kRowsAtOnce ? ((size_t)B + 1) * sizeof(int32_t) : 0;
}

extern "C" int moba_paged_reserve(int32_t* free_pages, int32_t* free_count, int32_t* page_table, int32_t* lengths,
                                  const int32_t* new_tokens, int32_t* cu_new, int32_t* owners, int32_t* positions, int64_t* slots,
                                  void* workspace, int B, int64_t rows, int page_size, int64_t num_pages, int64_t max_pages,
                                  int64_t table_stride, void* stream) {
  TableParams p;
  const int rc = check_tables(p, free_pages, free_count, page_table, lengths, new_tokens, B, page_size, num_pages, max_pages, table_stride);
  if (rc != MOBA_OK) return rc;
  if (!cu_new || rows < 0 || (rows > kRowsAtOnce && !workspace) || (rows && (!owners || !positions || !slots)) || ((uintptr_t)slots & 7) ||
      ((uintptr_t)workspace & 3))
    return MOBA_ERR_ARG;
  if (rows >= 1LL << 30) return MOBA_ERR_LIMIT;
  p.cu_new = cu_new; p.owners = owners; p.positions = positions; p.slots = slots; p.ranks = (int32_t*)workspace;
  p.rows = (int)rows;
  LaunchCheck launch_check;
  hipStream_t st = (hipStream_t)stream;
  const int need = (3 * B + 2) * 4;
  static bool allowed[2][kMaxDevices];
  if (!allow_dynamic_lds((const void*)paged_reserve_kernel, (3 * kMostTableSequences + 2) * 4, allowed[0]) ||
      !allow_dynamic_lds((const void*)paged_rows_kernel, (3 * kMostTableSequences + 2) * 4, allowed[1]))
    return MOBA_ERR_LAUNCH;
  hipLaunchKernelGGL(paged_reserve_kernel, dim3(1), dim3(kTableThreads), need, st, p);
  if (rows > kRowsAtOnce)
    hipLaunchKernelGGL(paged_rows_kernel, dim3((unsigned)((rows + 1023) / 1024)), dim3(256), need, st, p);
  return launch_check.result();
}

extern "C" int moba_paged_release(int32_t* free_pages, int32_t* free_count, int32_t* page_table, int32_t* lengths, const int32_t* keep,
                                  int B, int page_size, int64_t num_pages, int64_t max_pages, int64_t table_stride, void* stream) {
  TableParams p;
  const int rc = check_tables(p, free_pages, free_count, page_table, lengths, keep, B, page_size, num_pages, max_pages, table_stride);
  if (rc != MOBA_OK) return rc;
  LaunchCheck launch_check;
  static bool allowed[kMaxDevices];
  if (!allow_dynamic_lds((const void*)paged_release_kernel, 2 * kMostTableSequences * 4, allowed)) return MOBA_ERR_LAUNCH;
  hipLaunchKernelGGL(paged_release_kernel, dim3(1), dim3(kTableThreads), 2 * B * 4, (hipStream_t)stream, p);
  return launch_check.result();
}
