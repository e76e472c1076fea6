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
// One workgroup decides (the sums over the sequences, in LDS), fills the table and, for up to kRowsAtOnce rows, says where they belong;
// more rows are a second launch of as many workgroups as that takes.  Nothing here is floating point, and no order depends on
// timing: sums are scans.  Bound by latency: loads of the lengths, two scans, a search in LDS and a load for every page and row.
#include "common.h"
#include "paged.h"

namespace moba {

constexpr int kTableThreads = 1024, kTableWaves = kTableThreads / 64;
constexpr int kMostTableSequences = 8192;   // whose sums fit a workgroup's LDS
constexpr int kRowsAtOnce = 4096;
constexpr int kPagesOfThread = 8;           // that a thread moves at a time, where there are more than threads

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
  int64_t stride;
  int B, rows, max_pages, page_log2;
};

// inclusive sums over the threads up to this one, and over all of them.  `red`: [2 * kTableWaves]; every thread calls it
template <class T>
struct Scan {
  T upto, all;
};
template <class T>
__device__ __forceinline__ Scan<T> scan(T x, T* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  __syncthreads();   // (the former call's sums have been read)
  if (lane == 63) red[wave] = x;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kTableWaves; ++w) {
    const T y = red[w];
    before += w < wave ? y : 0;
    all += y;
  }
  return {x + before, all};
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

// Row t, whose sequence's rows are cu[b] .. cu[b+1] - 1 and end at its last token
__device__ __forceinline__ void place_row(const TableParams& p, const int* cu, int t) {
  int b = -1, position = 0;
  int64_t slot = -1;
  if (t < cu[p.B]) {
    b = last_at_most(cu, p.B, t);
    position = p.lengths[b] - (cu[b + 1] - t);
    const int page = position >> p.page_log2;
    const int id = position >= 0 && page < p.max_pages ? p.table[b * p.stride + page] : -1;
    if (id >= 0 && id < p.pool.num_pages) slot = ((int64_t)id << p.page_log2) + (position & ((1 << p.page_log2) - 1));
  }
  p.owners[t] = b;
  p.positions[t] = position;
  p.slots[t] = slot;
}

__global__ __launch_bounds__(kTableThreads) void paged_reserve_kernel(const TableParams p) {
  extern __shared__ __attribute__((aligned(8))) int lds[];
  int64_t* const red = reinterpret_cast<int64_t*>(lds);
  int* const rank = lds + 2 * kTableWaves;   // [B]: pages given to the sequences before
  int* const have = rank + p.B;              // [B]: pages that a sequence had
  int* const cu = have + p.B;                // [B+1]
  const int tid = threadIdx.x;
  const int free_count = min(max(*p.pool.free_count, 0), p.pool.num_pages);
  const int64_t most = min((int64_t)p.max_pages << p.page_log2, (int64_t)0x7fffffff);
  int64_t asked = 0, asked_pages = 0;   // sums over the sequences of the steps before
  int given = 0, given_pages = 0;
  for (int b0 = 0; b0 < p.B; b0 += kTableThreads) {
    const int b = b0 + tid;
    int64_t old = 0, n = 0;
    if (b < p.B) {
      old = max(p.lengths[b], 0);
      n = max(p.asked[b], 0);
      if (old + n > most) n = 0;
    }
    const int held = pages_of(old, p.page_log2), need = pages_of(old + n, p.page_log2) - held;
    const Scan<int64_t> tokens = scan<int64_t>(n, red), pages = scan<int64_t>(need, red);
    const bool served = asked + tokens.upto <= p.rows && (need == 0 || asked_pages + pages.upto <= free_count);
    asked += tokens.all;
    asked_pages += pages.all;
    // (of the served both sums fit 31 bits)
    const Scan<int64_t> both = scan<int64_t>(served ? n << 32 | need : 0, red);
    if (b < p.B) {
      cu[b + 1] = given + (int)(both.upto >> 32);
      rank[b] = given_pages + (int)(uint32_t)both.upto - (served ? need : 0);
      have[b] = held;
      p.cu_new[b + 1] = cu[b + 1];
      if (served && n) p.lengths[b] = (int)(old + n);
    }
    given += (int)(both.all >> 32);
    given_pages += (int)(uint32_t)both.all;
  }
  if (tid == 0) {
    cu[0] = 0;
    p.cu_new[0] = 0;
    *p.pool.free_count = free_count - given_pages;
  }
  __syncthreads();
  const int each = given_pages > kTableThreads ? kPagesOfThread : 1;
  for (int64_t i0 = (int64_t)tid * each; i0 < given_pages; i0 += kTableThreads * each) {
    int b = last_at_most(rank, p.B, (int)i0);
    for (int i = (int)i0; i < min(i0 + each, (int64_t)given_pages); ++i) {
      while (b + 1 < p.B && rank[b + 1] <= i) ++b;
      p.table[b * p.stride + have[b] + i - rank[b]] = p.pool.free_pages[free_count - 1 - i];
    }
  }
  if (p.rows > kRowsAtOnce) return;
  __syncthreads();   // (the table and the lengths are written)
  for (int t = tid; t < p.rows; t += kTableThreads) place_row(p, cu, t);
}

__global__ __launch_bounds__(256) void paged_rows_kernel(const TableParams p) {
  extern __shared__ __attribute__((aligned(8))) int cu[];
  for (int b = threadIdx.x; b <= p.B; b += 256) cu[b] = p.cu_new[b];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t t = (int64_t)blockIdx.x * 1024 + k * 256 + threadIdx.x;
    if (t < p.rows) place_row(p, cu, (int)t);
  }
}

__global__ __launch_bounds__(kTableThreads) void paged_release_kernel(const TableParams p) {
  extern __shared__ __attribute__((aligned(8))) int lds[];
  int64_t* const red = reinterpret_cast<int64_t*>(lds);
  int* const first = lds + 2 * kTableWaves;  // [B]: entries that go in the sequences before (their number is below 2^31)
  int* const stay = first + p.B;             // [B]: pages that stay
  const int tid = threadIdx.x;
  int free_count = min(max(*p.pool.free_count, 0), p.pool.num_pages), total = 0;
  for (int b0 = 0; b0 < p.B; b0 += kTableThreads) {
    const int b = b0 + tid;
    int gone = 0, kept = 0;
    if (b < p.B) {
      const int old = max(p.lengths[b], 0), keep = min(max(p.asked[b], 0), old);
      kept = min(pages_of(keep, p.page_log2), p.max_pages);
      gone = min(pages_of(old, p.page_log2), p.max_pages) - kept;
      if (keep < old) p.lengths[b] = keep;
    }
    const Scan<int64_t> s = scan<int64_t>(gone, red);
    if (b < p.B) {
      first[b] = total + (int)s.upto - gone;
      stay[b] = kept;
    }
    total += (int)s.all;
  }
  __syncthreads();
  // from the last entry to the first, so that a place on the stack is the number of pages that have come before
  const int each = total > kTableThreads ? kPagesOfThread : 1;
  for (int64_t r0 = 0; r0 < total; r0 += kTableThreads * each) {
    const int64_t mine = r0 + (int64_t)tid * each;
    int id[kPagesOfThread], count = 0;
    if (mine < total) {
      int b = last_at_most(first, p.B, total - 1 - (int)mine);
#pragma unroll
      for (int k = 0; k < kPagesOfThread; ++k) {
        id[k] = -1;
        if (k >= each || mine + k >= total) continue;
        const int i = total - 1 - (int)(mine + k);
        while (first[b] > i) --b;
        int32_t* const entry = p.table + b * p.stride + stay[b] + i - first[b];
        const int x = *entry;
        *entry = -1;
        if (x >= 0 && x < p.pool.num_pages) {
          id[k] = x;
          ++count;
        }
      }
    }
    const Scan<int64_t> s = scan<int64_t>(count, red);
    if (mine < total) {
      int64_t place = free_count + s.upto - count;
#pragma unroll
      for (int k = 0; k < kPagesOfThread; ++k)
        if (k < each && id[k] >= 0) {
          if (place < p.pool.num_pages) p.pool.free_pages[place] = id[k];   // (more than there are: named twice)
          ++place;
        }
    }
    free_count = (int)min(free_count + s.all, (int64_t)p.pool.num_pages);
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

extern "C" int moba_paged_reserve(int32_t* free_pages, int32_t* free_count, int32_t* page_table, int32_t* lengths,
                                  const int32_t* new_tokens, int32_t* cu_new, int32_t* owners, int32_t* positions, int64_t* slots, int B,
                                  int64_t rows, int page_size, int64_t num_pages, int64_t max_pages, int64_t table_stride, void* stream) {
  TableParams p;
  const int rc = check_tables(p, free_pages, free_count, page_table, lengths, new_tokens, B, page_size, num_pages, max_pages, table_stride);
  if (rc != MOBA_OK) return rc;
  if (!cu_new || rows < 0 || (rows && (!owners || !positions || !slots)) || ((uintptr_t)slots & 7)) return MOBA_ERR_ARG;
  if (rows >= 1LL << 30) return MOBA_ERR_LIMIT;
  p.cu_new = cu_new; p.owners = owners; p.positions = positions; p.slots = slots;
  p.rows = (int)rows;
  static bool allowed[kMaxDevices];
  const int most_lds = (2 * kTableWaves + 3 * kMostTableSequences + 1) * 4, need = (2 * kTableWaves + 3 * B + 1) * 4;
  LaunchCheck launch_check;
  if (!allow_dynamic_lds((const void*)paged_reserve_kernel, most_lds, allowed)) return MOBA_ERR_LAUNCH;
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(paged_reserve_kernel, dim3(1), dim3(kTableThreads), need, st, p);
  if (rows > kRowsAtOnce)
    hipLaunchKernelGGL(paged_rows_kernel, dim3((unsigned)((rows + 1023) / 1024)), dim3(256), (B + 1) * 4, st, p);
  return launch_check.result();
}

extern "C" int moba_paged_release(int32_t* free_pages, int32_t* free_count, int32_t* page_table, int32_t* lengths, const int32_t* keep,
                                  int B, int page_size, int64_t num_pages, int64_t max_pages, int64_t table_stride, void* stream) {
  TableParams p;
  const int rc = check_tables(p, free_pages, free_count, page_table, lengths, keep, B, page_size, num_pages, max_pages, table_stride);
  if (rc != MOBA_OK) return rc;
  static bool allowed[kMaxDevices];
  const int most_lds = (2 * kTableWaves + 2 * kMostTableSequences) * 4, need = (2 * kTableWaves + 2 * B) * 4;
  LaunchCheck launch_check;
  if (!allow_dynamic_lds((const void*)paged_release_kernel, most_lds, allowed)) return MOBA_ERR_LAUNCH;
  hipLaunchKernelGGL(paged_release_kernel, dim3(1), dim3(kTableThreads), need, (hipStream_t)stream, p);
  return launch_check.result();
}
