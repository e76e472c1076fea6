// The blocks of the paged cache that a new token attends: the sums of the pages' keys, kept up with the cache, and the blocks with the
// largest products with them (the reference's gate for whole prompts: moba/moba_efficient.py:326-371).
//
//   sum[page, h, :]   = sum over the tokens that the page holds of k[page, h, token, :], 32 bits
//   score[t, h, j]    = q[t, h, :] . sum over block j's pages of sum[page, h / rep, :], 64 bits
//   blocks[t, h, :]   = the topk - 1 blocks before the token's own with the largest scores (of equal ones the lowest), and its own;
//                       ascending, -1 behind the last
// Blocks before a token's own are whole, so that the order of the sums is that of the means.  In 64 bits a score is off by some 2^-53 of
// the sum of its terms' magnitudes for each of its additions; of scores nearer than that rounding decides, and always alike: a score is
// the result of the same operations in the same order whatever else is in the batch, and blocks of the same pages have equal scores.
//
// All three kernels are bound by memory or latency.
//   Sums       the keys of the pages that have received tokens, once: 131072 tokens, 8 heads, 8 bits: 143 MB in 30.4 us, 22.7 where they
//              are in the last-level cache; the next token of 16 sequences 3.6.
//   Scores     the sums of the history's pages once for up to 32 rows (tokens times heads) of a key/value head; a workgroup's threads
//              take 16 bytes of a page each, so that a whole block of many pages is on its way at once.  32 heads on 8, blocks of 4096
//              behind 131072: 8.0 us, 6.2 where the sums are in a cache; 16 sequences of five tokens, blocks of 512, 15 MB: 15.4 and 12.7.
//   Selection  the scores of a row stay in registers, as whole numbers in the same order, of which the (topk - 1)-th largest is found
//              bit by bit: a comparison and a count for each of a lane's scores and bit, until the count is right (some 20 bits).
//              3.8 and 5.4 us of these.
#include "attn_common.h"
#include "paged_cut.h"

namespace moba {

// ---- sums of keys
template <class E>
struct SumParams {
  PageTable table;
  const char* pages;
  const float* scales;   // 8-bit pages
  float* sums;           // [num_pages, Hkv, D]
  int64_t unit0;         // pages of the batch, numbered through, of this launch: the first,
  int Hkv, items;        // and how many times heads (waves)
};
constexpr int64_t kSumItems = (1 << 25) - 1;   // of a launch: below 2^31 threads

// One wave to a page and head: 64 / L tokens at a time, L lanes of 16 bytes to a token, kAhead such steps on their way together.  (Eight of
// them: 22.4 us for 131072 tokens as above, 22.7 so, but 8192 on pages of 16 6.3 and 5.0.  Two heads to a wave: 23.6 and 4.9, and the next
// token of 16 sequences 4.3.)
template <class E, int D, bool k8>
__global__ __launch_bounds__(256) void paged_key_sums_kernel(const SumParams<E> p) {
  constexpr int kRow = D * (k8 ? 1 : 2), L = kRow / 16, kTokens = 64 / L, kElems = k8 ? 16 : 8, kAhead = 4;
  const int lane = threadIdx.x & 63;
  const int item = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + (threadIdx.x >> 6));
  if (item >= p.items) return;
  const PageTable& table = p.table;
  const int unit = item / p.Hkv, hkv = item - unit * p.Hkv;
  const int64_t u = p.unit0 + unit;
  Sequence seq = {};
  auto start = [&](int b, int lo) { return (int64_t)(lo >> table.page_log2) + 2 * (int64_t)b; };
  const int b = last_up_to(table, u, lane, seq, start);
  if (b < 0 || seq.hi == seq.lo) return;
  const int64_t began = max(seq.length - (seq.hi - seq.lo), (int64_t)0);
  const int64_t page = (began >> table.page_log2) + (u - start(b, seq.lo));
  const int held = (int)min(max(seq.length - (page << table.page_log2), (int64_t)0), (int64_t)1 << table.page_log2);
  const int id = __builtin_amdgcn_readfirstlane(page_id(table, b, page));
  if (held == 0 || id < 0) return;
  const int r = lane / L, c = lane % L;
  const int64_t head = (int64_t)id * p.Hkv + hkv;
  const char* const from = p.pages + (head << table.page_log2) * kRow + c * 16;
  const float by = k8 ? p.scales[head] : 1.f;
  float acc[kElems];
#pragma unroll
  for (int e = 0; e < kElems; ++e) acc[e] = 0.f;
  for (int t0 = 0; t0 < held; t0 += kTokens * kAhead) {
    u32x4 w[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)   // (those behind the last held one are it again)
      w[k] = *reinterpret_cast<const u32x4*>(from + min(t0 + k * kTokens + r, held - 1) * kRow);
    if (t0 + kTokens * kAhead > held) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (t0 + k * kTokens + r >= held) w[k] = u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if constexpr (k8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[4 * i] += __builtin_amdgcn_cvt_f32_fp8(w[k][i], 0);
          acc[4 * i + 1] += __builtin_amdgcn_cvt_f32_fp8(w[k][i], 1);
          acc[4 * i + 2] += __builtin_amdgcn_cvt_f32_fp8(w[k][i], 2);
          acc[4 * i + 3] += __builtin_amdgcn_cvt_f32_fp8(w[k][i], 3);
        }
      } else {
        const typename E::elem8 x = __builtin_bit_cast(typename E::elem8, w[k]);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += (float)x[e];
      }
    }
  }
  // the lanes of a column: each keeps half of what it has and is given the other's of that half
  int at = c * kElems;
  auto halve = [&](auto step) __attribute__((always_inline)) {
    constexpr int m = 32 >> step, n = kElems >> (step + 1);
    if constexpr (m >= L) {
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const uint32_t x = float_bits(acc[i]), y = float_bits(acc[i + n]);
        uint32_t mine, other;   // what the lane has of its half, and what the other one has
        if constexpr (m == 32) {
          const auto z = __builtin_amdgcn_permlane32_swap(x, y, false, false);
          mine = z[0], other = z[1];
        } else if constexpr (m == 16) {
          const auto z = __builtin_amdgcn_permlane16_swap(x, y, false, false);
          mine = z[0], other = z[1];
        } else {
          // (a choice of bits: one of elements becomes one of their numbers, and a search among all: 5.9 us for 16 sequences' next tokens)
          const uint32_t upper = -(uint32_t)((lane & m) != 0);
          mine = (x & ~upper) | (y & upper);
          other = (uint32_t)__shfl_xor((int)((x & upper) | (y & ~upper)), m, 64);
        }
        acc[i] = __builtin_bit_cast(float, mine) + __builtin_bit_cast(float, other);
      }
      at += lane & m ? n : 0;
    }
  };
  halve(std::integral_constant<int, 0>{});
  halve(std::integral_constant<int, 1>{});
  halve(std::integral_constant<int, 2>{});
  halve(std::integral_constant<int, 3>{});
#pragma unroll
  for (int i = 0; i < D / 64; ++i) p.sums[head * D + at + i] = acc[i] * by;
}

// ---- scores
constexpr int kScoreRows = 32, kScoreSumsLog2 = 4, kScoreSums = 1 << kScoreSumsLog2;
constexpr int kMostBlocks = 16384;   // of a sequence

struct SelectShape {
  PageTable table;
  int H, Hkv, rep;
  int each;             // pages of a block
  int blocks;           // that a row of the table has room for
  int topk;
  int t0, tokens;       // rows of this launch
};
template <class E>
struct SelectParams {
  SelectShape s;
  const typename E::elem* q;
  int64_t q_tok_stride, q_head_stride;
  const float* sums;
  double* scores;       // [tokens, H, blocks]
  int split_log2;       // sums that a block's pages are shared out to
};
__device__ __forceinline__ int64_t block_tokens(const SelectShape& s) { return (int64_t)s.each << s.table.page_log2; }

// A workgroup forms the sums of up to 16 blocks (fewer where a block's pages are shared out among threads) in LDS, and their products
// with its rows by v_mfma_f64_16x16x4, a quarter of the elements to a wave.
template <class E, int D>
__global__ __launch_bounds__(256) void paged_score_kernel(const SelectParams<E> p) {
  constexpr int kQuads = D / 4, kThreads = 256 / kQuads, kRounds = kScoreSums / kThreads, kAhead = 4;
  typedef double f64x4 __attribute__((ext_vector_type(4)));
  __shared__ double part[kScoreSums][D + 2];
  __shared__ float rows[kScoreRows][D + 4];
  __shared__ double red[4][kScoreRows][kScoreSums + 1];
  const SelectShape& s = p.s;
  const PageTable& table = s.table;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hkv = blockIdx.y;
  Sequence seq = {};
  auto cut = [&](int row) { return min(max(row - s.t0, 0), s.tokens); };
  auto start = [&](int b, int lo) { return (int64_t)cut(lo) * s.rep / kScoreRows + b; };
  const int b = last_up_to(table, blockIdx.x, lane, seq, start);
  if (b < 0) return;
  const int lo = cut(seq.lo) + s.t0, hi = cut(seq.hi) + s.t0;   // the sequence's rows of this launch
  const int64_t row0 = ((int64_t)blockIdx.x - start(b, seq.lo)) * kScoreRows, count = (int64_t)(hi - lo) * s.rep;
  if (row0 >= count) return;
  const int rows_here = (int)min(count - row0, (int64_t)kScoreRows);
  const int64_t last = seq.length - seq.hi + lo + (row0 + rows_here - 1) / s.rep;   // position of the last of them
  const int history = (int)min(max(last, (int64_t)0) / block_tokens(s), (int64_t)s.blocks);
  const int split = 1 << p.split_log2, at_once = kScoreSums >> p.split_log2;
  if ((int)blockIdx.z * at_once >= history) return;
  for (int i = tid; i < rows_here * (D / 8); i += 256) {
    const int r = i / (D / 8), d = i % (D / 8) * 8, row = (int)row0 + r, j = row / s.rep;
    const typename E::elem8 x = *reinterpret_cast<const typename E::elem8*>(p.q + (int64_t)(lo + j) * p.q_tok_stride +
                                                                           (int64_t)(hkv * s.rep + row - j * s.rep) * p.q_head_stride + d);
#pragma unroll
    for (int e = 0; e < 8; ++e) rows[r][d + e] = (float)x[e];
  }
  const int quad = tid % kQuads;
  for (int j0 = blockIdx.z * at_once; j0 < history; j0 += gridDim.z * at_once) {
    // Sum number i: of block i % at_once, its pages i / at_once, .. + split, ..  Whatever the split, pages that are half as many apart as
    // the block has places for (its pages, rounded up to a power of two) are added first, then sums that are a quarter apart, and so on
    // (of blocks of more than 64 pages, which are always split alike, those 64 apart first): a thread's sums by their distance,
    // then those of the threads.  (Sums whose order the split decides: single tokens of 256 sequences, 8 pages to a block, 43.2 us, 44.3 so.)
    double acc[kRounds][kAhead][4];
    auto add_pages = [&](int i0, auto first) __attribute__((always_inline)) {
      f32x4 x[kRounds][kAhead];
#pragma unroll
      for (int k = 0; k < kRounds; ++k) {
        const int sum = tid / kQuads + k * kThreads, j = j0 + (sum & (at_once - 1));
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
          const int i = i0 + a * split + (sum >> (kScoreSumsLog2 - p.split_log2));
          const int id = i < s.each && j < history ? page_id(table, b, (int64_t)j * s.each + i) : -1;
          x[k][a] = f32x4{0.f, 0.f, 0.f, 0.f};
          if (id >= 0) x[k][a] = *reinterpret_cast<const f32x4*>(p.sums + ((int64_t)id * s.Hkv + hkv) * D + 4 * quad);
        }
      }
#pragma unroll
      for (int k = 0; k < kRounds; ++k)
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[k][a][e] = first ? (double)x[k][a][e] : acc[k][a][e] + (double)x[k][a][e];
    };
    add_pages(0, std::true_type{});
    for (int i0 = split * kAhead; i0 < s.each; i0 += split * kAhead) add_pages(i0, std::false_type{});
    static_assert(kAhead == 4);
#pragma unroll
    for (int k = 0; k < kRounds; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        part[tid / kQuads + k * kThreads][4 * quad + e] = (acc[k][0][e] + acc[k][2][e]) + (acc[k][1][e] + acc[k][3][e]);
    __syncthreads();
    auto join = [&](auto log2) __attribute__((always_inline)) {
      constexpr int kSplit = 1 << log2, kBlocks = kScoreSums / kSplit;
      for (int i = tid; i < kBlocks * D; i += 256) {
        double x[kSplit];
#pragma unroll
        for (int k = 0; k < kSplit; ++k) x[k] = part[k * kBlocks + i / D][i % D];
#pragma unroll
        for (int h = kSplit / 2; h >= 1; h /= 2)
#pragma unroll
          for (int k = 0; k < h; ++k) x[k] += x[k + h];
        part[i / D][i % D] = x[0];
      }
      __syncthreads();
    };
    static_assert(kScoreSumsLog2 == 4);
    if (p.split_log2 == 1) join(std::integral_constant<int, 1>{});
    else if (p.split_log2 == 2) join(std::integral_constant<int, 2>{});
    else if (p.split_log2 == 3) join(std::integral_constant<int, 3>{});
    else if (p.split_log2 == 4) join(std::integral_constant<int, 4>{});
    // (rows and blocks that are none have columns and rows of their own)
    for (int r0 = 0; r0 < rows_here; r0 += 16) {
      f64x4 c = {0., 0., 0., 0.};
#pragma unroll
      for (int m = 0; m < D / 16; ++m) {
        const int d = wave * (D / 4) + 4 * m + (lane >> 4);
        c = __builtin_amdgcn_mfma_f64_16x16x4f64((double)rows[r0 + (lane & 15)][d], part[lane & 15][d], c, 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) red[wave][r0 + (lane >> 4) + 4 * e][lane & 15] = c[e];
    }
    __syncthreads();
    for (int r = tid >> 4; r < rows_here; r += 16) {
      const int j = tid & 15, row = (int)row0 + r, t = row / s.rep;
      if (j < at_once && j0 + j < history)
        p.scores[((int64_t)(lo - s.t0 + t) * s.H + hkv * s.rep + row - t * s.rep) * s.blocks + j0 + j] =
            red[0][r][j] + red[1][r][j] + red[2][r][j] + red[3][r][j];
    }
  }
}

// ---- selection
// a score as a whole number, in the same order; NaN is the least, with minus infinity
__device__ __forceinline__ uint64_t in_order(double x) {
  if (x != x) x = -INFINITY;
  const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.);   // (one zero)
  return u >> 63 ? ~u : u | 1ull << 63;
}

struct PickParams {
  SelectShape s;
  const double* scores;
  int32_t* out;         // [T, H, topk]
  int64_t row0;         // of this launch, among the rows (tokens times heads) that have scores
};

// A row for kWaves waves, kPer scores to a lane: block i * 64 * kWaves + thread is register i of a thread
template <int kWaves, int kPer>
__global__ __launch_bounds__(kWaves == 1 ? 256 : 64 * kWaves) void paged_pick_kernel(const PickParams p) {
  constexpr int kThreads = 64 * kWaves;
  __shared__ int counts[2][kWaves], places[kPer * kWaves];
  const SelectShape& s = p.s;
  const int lane = threadIdx.x & 63, wave = kWaves == 1 ? 0 : threadIdx.x >> 6, tid = kWaves == 1 ? lane : threadIdx.x;
  const int64_t row = p.row0 + (kWaves == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x);
  if (row >= (int64_t)s.tokens * s.H) return;
  const int t = s.t0 + (int)(row / s.H);
  int32_t* const out = p.out + ((int64_t)s.t0 * s.H + row) * s.topk;
  Sequence seq = {};
  const int b = last_up_to(s.table, t, lane, seq, [](int, int lo) { return (int64_t)lo; });
  const int64_t position = b >= 0 && t < seq.hi ? seq.length - seq.hi + t : -1;
  const int64_t own = position >= 0 ? position / block_tokens(s) : s.blocks;
  const int history = position >= 0 ? (int)min(own, (int64_t)s.blocks) : 0, picks = min(s.topk - 1, history);
  uint64_t key[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int j = i * kThreads + tid;
    key[i] = 0;   // (less than any score's)
    if (picks < history && j < history) key[i] = in_order(p.scores[row * s.blocks + j]);
  }
  int parity = 0;
  auto total = [&](int mine) __attribute__((always_inline)) {   // the sum over the waves
    if constexpr (kWaves == 1) return mine;
    if (lane == 0) counts[parity][wave] = mine;
    __syncthreads();
    int x = lane < kWaves ? counts[parity][lane] : 0;
    parity ^= 1;
    return (int)wave_sum((uint32_t)x);
  };
  // in `before`: of the blocks that have bit i of `in` in ascending order, how many lie before this thread's first of register i;
  // their number
  auto number = [&](uint32_t in, int (&before)[kPer]) __attribute__((always_inline)) {
    int all = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint64_t m = __ballot(in >> i & 1);
      before[i] = __builtin_popcountll(m & ((1ull << lane) - 1));
      if constexpr (kWaves == 1) {
        before[i] += all;
        all += __builtin_popcountll(m);
      } else if (lane == 0) {
        places[i * kWaves + wave] = __builtin_popcountll(m);
      }
    }
    if constexpr (kWaves > 1) {
      constexpr int kEach = kPer * kWaves / 64;
      __syncthreads();
      int x[kEach], sum = 0;
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        x[k] = places[lane * kEach + k];
        sum += x[k];
      }
      const int upto = (int)upto_sum((uint32_t)sum);
      all = __builtin_amdgcn_readlane(upto, 63);
      __syncthreads();
      if (wave == 0) {
        int at = upto - sum;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
          places[lane * kEach + k] = at;
          at += x[k];
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPer; ++i) before[i] += places[i * kWaves + wave];
      __syncthreads();   // (`places` has been read)
    }
    return all;
  };
  uint32_t chosen = 0;   // bit i: register i
  int before[kPer];
  if (picks == history) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) chosen |= (uint32_t)(i * kThreads + tid < history) << i;
  } else if (picks > 0) {
    uint64_t least = 0;   // of the chosen, from its highest bit on
    bool exact = false;
    for (int bit = 63; bit >= 0 && !exact; --bit) {
      const uint64_t to = least | 1ull << bit;
      int mine = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) mine += __builtin_popcountll(__ballot(key[i] >= to));
      const int n = total(mine);
      if (n >= picks) least = to;
      exact = n == picks;
    }
    uint32_t same = 0;
    int above = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool in = exact ? key[i] >= least : key[i] > least;
      chosen |= (uint32_t)in << i;
      same |= (uint32_t)(key[i] == least) << i;
      above += __builtin_popcountll(__ballot(in));
    }
    if (!exact) {   // equal scores: the lowest blocks
      const int left = picks - total(above);
      number(same, before);
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if ((same >> i & 1) && before[i] < left) chosen |= 1u << i;
    }
  }
  const int count = number(chosen, before);
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (chosen >> i & 1) out[before[i]] = i * kThreads + tid;
  if (tid < s.topk && tid >= count) out[tid] = tid == count && own < s.blocks ? (int)own : -1;
}

static constexpr int64_t kScoreBytes = 1LL << 29;   // of a launch's scores: more tokens are several launches
constexpr int64_t kPickRows = 1LL << 21;            // of a launch: below 2^32 threads for up to sixteen waves to a row
constexpr int kMostTopk = 64;

static int blocks_of(int64_t max_pages, int each) { return (int)((max_pages + each - 1) / each); }
static int64_t tokens_at_once(int64_t T, int H, int blocks) {
  const int64_t n = kScoreBytes / ((int64_t)H * blocks * 8);
  return n < 1 ? 1 : n < T ? n : T;
}

template <class E, int D>
static int launch_select(SelectParams<E> p, int32_t* out, int64_t T, hipStream_t st) {
  LaunchCheck launch_check;
  SelectShape& s = p.s;
  const int64_t step = tokens_at_once(T, s.H, s.blocks);
  for (int64_t t0 = 0; t0 < T; t0 += step) {
    s.t0 = (int)t0;
    s.tokens = (int)(T - t0 < step ? T - t0 : step);
    const int64_t units = (int64_t)s.tokens * s.rep / kScoreRows + s.table.B;
    // (a thread has up to eight pages of a block on its way; fewer where there are not enough blocks for the chip.  Blocks of 64 pages behind
    // 131072 tokens 6.2 us, 7.5 without the latter, 30 with a thread to a block; of 8 pages behind 20000 5.0 and 7.2.  Up to four, two and one
    // page to a thread wherever a block has several, the whole call: 16 sequences of five tokens, 8 pages to a block, 19, 22 and 32 us, 16.5
    // so; 2048 tokens behind 131072, 64 pages, 588, 455 so)
    auto chunks = [&]() { return (s.blocks - 1) / (kScoreSums >> p.split_log2) + 1; };
    p.split_log2 = 0;
    while (p.split_log2 < kScoreSumsLog2 &&
           (s.each > 8 << p.split_log2 || (s.each > 1 << p.split_log2 && units * s.Hkv * chunks() < 512)))
      ++p.split_log2;
    const int64_t want = 4096 / (units * s.Hkv);
    const int z = (int)(want < 1 ? 1 : want < chunks() ? want : chunks());
    hipLaunchKernelGGL((paged_score_kernel<E, D>), dim3((unsigned)units, s.Hkv, z), dim3(256), 0, st, p);
    const int64_t rows = (int64_t)s.tokens * s.H;
    for (int64_t row0 = 0; row0 < rows; row0 += kPickRows) {
      const PickParams pick = {s, p.scores, out, row0};
      const int64_t here = rows - row0 < kPickRows ? rows - row0 : kPickRows;
      const dim3 four((unsigned)((here + 3) / 4));
      if (s.blocks <= 64) hipLaunchKernelGGL((paged_pick_kernel<1, 1>), four, dim3(256), 0, st, pick);
      else if (s.blocks <= 256) hipLaunchKernelGGL((paged_pick_kernel<1, 4>), four, dim3(256), 0, st, pick);
      else if (s.blocks <= 1024) hipLaunchKernelGGL((paged_pick_kernel<1, 16>), four, dim3(256), 0, st, pick);
      else hipLaunchKernelGGL((paged_pick_kernel<16, 16>), dim3((unsigned)here), dim3(1024), 0, st, pick);
    }
  }
  return launch_check.result();
}

static bool index_ok(const int32_t* page_table, const int32_t* lengths, const int32_t* cu_new, int64_t T, int B, int Hkv, int64_t num_pages,
                     int64_t max_pages) {
  return page_table && lengths && cu_new && T > 0 && B > 0 && Hkv > 0 && num_pages > 0 && max_pages > 0;
}
static PageTable table_of(const int32_t* page_table, const int32_t* lengths, const int32_t* cu_new, int64_t stride, int64_t T, int B,
                          int64_t num_pages, int64_t max_pages, int page_log2) {
  const int64_t reachable = 0x7fff0000LL >> page_log2;
  return {page_table, lengths, cu_new, stride, B, (int)T, (int)num_pages, (int)(max_pages < reachable ? max_pages : reachable), page_log2};
}

}  // namespace moba

using namespace moba;

extern "C" int moba_paged_key_sums(const void* k_pages, const float* k_scales, float* sums, const int32_t* page_table,
                                   const int32_t* lengths, const int32_t* cu_new, int64_t T, int B, int Hkv, int D, int page_size,
                                   int64_t num_pages, int64_t max_pages, int64_t table_stride, int cache8, int dtype, void* stream) {
  if (!k_pages || !sums || !index_ok(page_table, lengths, cu_new, T, B, Hkv, num_pages, max_pages) || (cache8 && !k_scales)) return MOBA_ERR_ARG;
  const int page_log2 = page_log2_of(page_size);
  if ((D != 64 && D != 128) || page_log2 < 0 || (dtype != MOBA_DTYPE_BF16 && dtype != MOBA_DTYPE_F16)) return MOBA_ERR_UNSUPPORTED;
  if (((uintptr_t)k_pages & 15) || ((uintptr_t)sums & 3)) return MOBA_ERR_ARG;
  const int64_t units = (T >> page_log2) + 2 * (int64_t)B;   // (sequence b's pages are numbered from (its first row / page_size) + 2b on)
  if (T >= 1LL << 30 || num_pages >= 1LL << 31 || max_pages >= 1LL << 31 || (int64_t)B * Hkv >= 1LL << 24) return MOBA_ERR_LIMIT;
  LaunchCheck launch_check;
  auto launch = [&](auto e, auto d, auto c8) {
    typedef decltype(e) E;
    SumParams<E> p = {table_of(page_table, lengths, cu_new, table_stride, T, B, num_pages, max_pages, page_log2), (const char*)k_pages,
                      k_scales, sums, 0, Hkv, 0};
    const int64_t step = kSumItems / Hkv;
    for (; p.unit0 < units; p.unit0 += step) {
      p.items = (int)(units - p.unit0 < step ? units - p.unit0 : step) * Hkv;
      const dim3 grid((unsigned)((p.items + 3) / 4));
      hipLaunchKernelGGL((paged_key_sums_kernel<E, d, c8>), grid, dim3(256), 0, (hipStream_t)stream, p);
    }
  };
  constexpr std::integral_constant<int, 64> d64;
  constexpr std::integral_constant<int, 128> d128;
  if (cache8) D == 128 ? launch(Bf16{}, d128, std::true_type{}) : launch(Bf16{}, d64, std::true_type{});
  else if (dtype == MOBA_DTYPE_F16) D == 128 ? launch(F16{}, d128, std::false_type{}) : launch(F16{}, d64, std::false_type{});
  else D == 128 ? launch(Bf16{}, d128, std::false_type{}) : launch(Bf16{}, d64, std::false_type{});
  return launch_check.result();
}

static int select_sizes(int64_t T, int B, int H, int Hkv, int page_size, int64_t max_pages, int block_size, int* each) {
  if (T <= 0 || B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || max_pages <= 0) return MOBA_ERR_ARG;
  if (page_log2_of(page_size) < 0 || block_size <= 0 || block_size % page_size) return MOBA_ERR_UNSUPPORTED;
  *each = block_size / page_size;
  if (T >= 1LL << 24 || T * H >= 1LL << 31 || max_pages >= 1LL << 31 || blocks_of(max_pages, *each) > kMostBlocks) return MOBA_ERR_LIMIT;
  return MOBA_OK;
}

extern "C" size_t moba_paged_select_blocks_workspace_bytes(int64_t T, int B, int H, int Hkv, int page_size, int64_t max_pages,
                                                           int block_size) {
  int each;
  if (select_sizes(T, B, H, Hkv, page_size, max_pages, block_size, &each) != MOBA_OK) return 0;
  const int blocks = blocks_of(max_pages, each);
  return (size_t)tokens_at_once(T, H, blocks) * H * blocks * sizeof(double);
}

// strides, in elements: {q token, q head, page table row}
extern "C" int moba_paged_select_blocks(const void* q, const float* sums, int32_t* blocks, const int32_t* page_table, const int32_t* lengths,
                                        const int32_t* cu_new, void* workspace, int64_t T, int B, int H, int Hkv, int D, int page_size,
                                        int64_t num_pages, int64_t max_pages, int block_size, int topk, const int64_t* strides, int dtype,
                                        void* stream) {
  if (!q || !sums || !blocks || !workspace || !strides || !index_ok(page_table, lengths, cu_new, T, B, Hkv, num_pages, max_pages) || topk <= 0)
    return MOBA_ERR_ARG;
  int each;
  const int rc = select_sizes(T, B, H, Hkv, page_size, max_pages, block_size, &each);
  if (rc != MOBA_OK) return rc;
  if ((D != 64 && D != 128) || (dtype != MOBA_DTYPE_BF16 && dtype != MOBA_DTYPE_F16)) return MOBA_ERR_UNSUPPORTED;
  if (((uintptr_t)q & 15) || ((uintptr_t)sums & 15) || ((uintptr_t)workspace & 7) || (strides[0] & 7) || (strides[1] & 7)) return MOBA_ERR_ARG;
  if (num_pages >= 1LL << 31 || topk > kMostTopk || Hkv > 65535) return MOBA_ERR_LIMIT;
  const int page_log2 = page_log2_of(page_size);
  const SelectShape shape = {table_of(page_table, lengths, cu_new, strides[2], T, B, num_pages, max_pages, page_log2), H, Hkv, H / Hkv, each,
                             blocks_of(max_pages, each), topk, 0, 0};
  const int64_t step = tokens_at_once(T, H, shape.blocks), units = step * shape.rep / kScoreRows + B;
  if (units * Hkv * 256 >= 1LL << 32) return MOBA_ERR_LIMIT;
  auto launch = [&](auto e) {
    typedef decltype(e) E;
    const SelectParams<E> p = {shape, (const typename E::elem*)q, strides[0], strides[1], sums, (double*)workspace, 0};
    return D == 128 ? launch_select<E, 128>(p, blocks, T, (hipStream_t)stream) : launch_select<E, 64>(p, blocks, T, (hipStream_t)stream);
  };
  return dtype == MOBA_DTYPE_F16 ? launch(F16{}) : launch(Bf16{});
}
