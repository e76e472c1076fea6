// Attention of new tokens over the paged cache: every new token against its sequence's keys up to itself, sequences of any
// lengths and any numbers of new tokens in one call, grouped-query heads in place.
//
// Few rows (paged_few_kernel): bound by memory, K and V of the cache are read once for up to 32 query rows of a key/value
// head.  The rows are the columns of matrix products (S^T = K Q^T, O^T += V^T P^T with v_mfma_f32_32x32x16), the four waves
// of a workgroup take different keys; a wave copies its own 32-key blocks of K and V global -> LDS, two stages, without
// barriers.  An 8-bit block is half the bytes of a 16-bit one, so two workgroups fit a compute unit where one does there;
// its elements become bf16 (K: the queries' type), which holds every e4m3 number, on the way from LDS to the products:
//   K  16 bytes of a key's row are two operands of eight elements (the order of a product's terms is free, and the
//      queries' operands take the same)
//   V  ds_read_b64_tr_b8 transposes 8 keys x 16 elements
// A page's key scale multiplies the scores, its value scale the probabilities, both in 32 bits.  One token of 32 heads on 8
// against 131072 keys in 8 bits: 268 MB in 47 us, 5.7 TB/s; 16 sequences of up to 24001 keys in fp16 on 8 bits: 128 MB in
// 26.8; four times five tokens against 12345 to 20480 keys in 16 bits: 294 MB in 51, 5.8 TB/s; one token against 4096
// keys: 7.6, most of it finding the unit, the pages, and the first copies.
//
// Precision: the scores' products are exact, their sums 32 bits.  With few rows a probability (times the value scale) goes to the second
// product as the sum of two elements, its rounded value and the rounded rest (16 bits of it in bf16, 22 in fp16): the products are not
// what bounds that kernel.  With many rows they are, and it is one element where queries and products have one type (ProbParts).
//
// Rows that see no key are zeros.  Values that are not finite reach the rows that see them and no others: a key that a row
// does not see has the probability 0, but 0 * Inf is NaN, so a wave whose sums are not finite goes through its keys again
// one by one, every row with the keys that it sees.  (Rows of a page behind the sequence's end are cleared on the way: they
// hold whatever was there.)
//
//   paged_few_kernel    one run of keys: out itself; several: the run's rows (normalised) and their log-sum-exps (base 2)
//   paged_many_kernel   the same for sequences of more rows
//   paged_merge_kernel  the runs of a row together; zeros where there is nothing to see
//
// Table says what a sequence attends: PageTable all of its keys, SharedTable (paged_shared.h) what it has in common with its neighbours
// together with them, ChosenTable (paged_chosen.h) some blocks.
#pragma once
#include "attn_common.h"
#include "paged_cut.h"
#include <algorithm>
#include <type_traits>

namespace moba {

constexpr int kFewWaves = 4;
constexpr int kFewKeys = 32;                       // of a wave's step
constexpr int kFewRows = 32;
constexpr int kFewTile = kFewWaves * kFewKeys;     // keys of a workgroup's step
constexpr int kSlot = 16;                          // keys of which a block's page is looked up together
constexpr int kBatch = 64 / (kFewKeys / kSlot);    // steps whose pages one wave looks up at a time
constexpr int kScaleBytes = 2 * 2 * 64 * 4;        // of a wave: two batches, K's and V's scales of 64 slots

template <class E, class Table = PageTable>
struct PagedParams {
  typedef typename E::elem elem;
  Shape<Table> shape;
  Cut few, many;
  const elem* q;
  elem* out;              // [T, H, D]
  const char* pages[2];
  const float* scales[2];
  float *few_o, *few_lse, *many_o, *many_lse;  // [parts * Hkv, group_rows, D] and [.., group_rows]
  Runs* runs;             // [B]
  int64_t q_tok_stride, q_head_stride;
  float scale_log2;
};

// 16-byte column in LDS of column c of a row of kRowBytes: 16 neighbouring rows at one column, 8 of 4 + 4 neighbouring rows at
// one column, and 4 rows at two columns each lie in different banks
template <int kRowBytes>
__device__ __forceinline__ int swizzled(int row, int c) {
  if constexpr (kRowBytes == 256) return c ^ ((row & 3) << 2) ^ ((row >> 2) & 3);
  else if constexpr (kRowBytes == 128) return c ^ (((row >> 1) & 3) << 1) ^ ((row >> 3) & 1);
  else return c ^ ((row >> 2) & 3);
}

// eight e4m3 numbers as elements of a 16-bit type (exact), for bf16 also times the power of two in `by` (its exponent; the
// instruction leaves out the rest of it)
__device__ __forceinline__ bf16x8 widened(uint32_t a, uint32_t b, Bf16, float by = 1.f) {
  const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, by, false), q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, by, true);
  const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, by, false), s = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, by, true);
  return bf16x8{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}
__device__ __forceinline__ f16x8 widened(uint32_t a, uint32_t b, F16) {
  const f16x2 p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, false), q = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, true);
  const f16x2 r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, false), s = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, true);
  return f16x8{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}

// ... times any other factor, rounded
__device__ __forceinline__ bf16x8 widened_by(uint32_t a, uint32_t b, float by) {
  const u32x4 w = {pack2<Bf16>(__builtin_amdgcn_cvt_f32_fp8(a, 0) * by, __builtin_amdgcn_cvt_f32_fp8(a, 1) * by),
                   pack2<Bf16>(__builtin_amdgcn_cvt_f32_fp8(a, 2) * by, __builtin_amdgcn_cvt_f32_fp8(a, 3) * by),
                   pack2<Bf16>(__builtin_amdgcn_cvt_f32_fp8(b, 0) * by, __builtin_amdgcn_cvt_f32_fp8(b, 1) * by),
                   pack2<Bf16>(__builtin_amdgcn_cvt_f32_fp8(b, 2) * by, __builtin_amdgcn_cvt_f32_fp8(b, 3) * by)};
  return __builtin_bit_cast(bf16x8, w);
}
__device__ __forceinline__ bool power_of_two(float x) {   // (a normal one, not negative)
  const uint32_t bits = float_bits(x);
  return !(bits & 0x807fffff) && bits - 1 < 0x7f7fffff;
}

// fp16 probabilities are kept 2^7 times larger (the running maximum may lag by 2^8: they stay below 2^15), so that
// those far below the maximum stay above the type's smallest number; the factor cancels
template <class V> struct ProbShift { static constexpr float value = 0.f; };
template <> struct ProbShift<F16> { static constexpr float value = 7.f; };
constexpr float kMaxLag = 8.f;
constexpr float kNoMax = -3e38f;  // before the first visible key (finite: exp2(m - m_new) stays defined)

// A wave's keys again, one after the other, in 32 bits and relative to the exact maximum, every row with the keys that it
// sees only: blocks of 32 keys from key_lo on, `step` apart, up to key_hi; look(key, sees): a key's page, or -1, and whether the
// lane's row sees it.  kSplit: the operands' order of elements is that of 16 bytes of e4m3 to two operands.  Leaves the sum of
// exponentials in the lower half of the wave.
template <class E, class V, int D, bool k8, bool kSplit, class Table, class Look>
__device__ __forceinline__ void one_by_one(const PagedParams<E, Table>& p, int hkv, int key_lo, int step, int key_hi, Look look,
                                           float scale, const typename E::elem8 (&bq)[D / 16], f32x16 (&oacc)[D / 32], float& m_run,
                                           float& l_run) {
  typedef typename E::elem8 elem8;
  typedef typename E::elem4 elem4;
  constexpr int kRowBytes = D * (k8 ? 1 : 2);
  const int hh = (threadIdx.x & 63) >> 5;
  const auto& shape = p.shape;
  const auto& table = shape.table;
  const int64_t page_bytes = ((int64_t)shape.Hkv << table.page_log2) * kRowBytes;
  const int64_t head_bytes = ((int64_t)hkv << table.page_log2) * kRowBytes;
  const int page_mask = (1 << table.page_log2) - 1;
  auto each_key = [&](auto use) __attribute__((always_inline)) {
    for (int key0 = key_lo; key0 < key_hi; key0 += step) {
      for (int key = key0; key < min(key0 + 32, key_hi); ++key) {
        bool sees;
        const int id = __builtin_amdgcn_readfirstlane(look(key, sees));
        if (id < 0) continue;
        const int64_t at = head_bytes + id * page_bytes + (key & page_mask) * kRowBytes;
        float d = 0.f, ks = 1.f, vs = 1.f;
        if constexpr (k8) {
          ks = p.scales[0][(int64_t)id * shape.Hkv + hkv];
          vs = p.scales[1][(int64_t)id * shape.Hkv + hkv];
        }
#pragma unroll
        for (int s8 = 0; s8 < D / 16; ++s8) {
          elem8 x;
          if constexpr (k8) {
            const u32x2 w = *reinterpret_cast<const u32x2*>(p.pages[0] + at +
                                                            (kSplit ? 32 * (s8 >> 1) + 16 * hh + 8 * (s8 & 1) : 16 * s8 + 8 * hh));
            x = widened(w[0], w[1], E{});
          } else {
            x = *reinterpret_cast<const elem8*>(p.pages[0] + at + (16 * s8 + 8 * hh) * 2);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) d += (float)bq[s8][e] * (float)x[e];
        }
        const float sc = sum_xhalf(d) * (scale * ks);
        if (sees) use(at, sc, vs);
      }
    }
  };
  m_run = kNoMax;
  each_key([&](int64_t, float sc, float) __attribute__((always_inline)) { m_run = fmaxf(m_run, sc); });
  const float ref = m_run - ProbShift<V>::value;
  float l = 0.f;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) oacc[db][e] = 0.f;
  each_key([&](int64_t at, float sc, float vs) __attribute__((always_inline)) {
    float pe = fast_exp2(sc - ref);
    l += pe;
    pe *= vs;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {   // (elements 8i + 4hh .. + 3)
      float x[4];
      if constexpr (k8) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p.pages[1] + at + 8 * i + 4 * hh);
        x[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
        x[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
        x[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
        x[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
      } else {
        const elem4 w = *reinterpret_cast<const elem4*>(p.pages[1] + at + (8 * i + 4 * hh) * 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (float)w[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) oacc[i >> 2][4 * (i & 3) + e] += pe * x[e];
    }
  });
  l_run = hh == 0 ? l : 0.f;
}

__device__ __forceinline__ float lane_value(float x, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane((int)float_bits(x), lane));
}

// two numbers, each as the sum of two elements: rounded, and the rounded rest
template <class V>
__device__ __forceinline__ void in_two(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack2<V>(a, b);
  asm("" : "+v"(hi));  // (not rounded once more, one by one, for the rests)
  const typename V::elem2 h = __builtin_bit_cast(typename V::elem2, hi);
  lo = pack2<V>(a - (float)h[0], b - (float)h[1]);
}

template <class Table>
constexpr int few_sets(int D) { return kShares<Table> && D == 64 ? 2 : 1; }
template <int D, bool k8>
constexpr int few_stage_bytes() { return 2 * kFewKeys * D * (k8 ? 1 : 2); }  // K and V of a step
constexpr int kListBytes = 8192;   // kChooses: a list that stays in LDS, behind the rest
template <int D, bool k8>
constexpr int few_list_at() {
  const int loop = kFewWaves * (2 * few_stage_bytes<D, k8>() + kScaleBytes);
  const int end = kFewWaves * (32 * (D + 4) * 4 + 2 * 32 * 4);
  return loop > end ? loop : end;
}
template <int D, bool k8, class Table>
constexpr int few_lds_bytes() { return few_list_at<D, k8>() + (kChooses<Table> ? kListBytes : 0); }

// Position of new token j of a unit's rows, every lane its own (mine: the lane's sequence of find_unit()); the least of a wave's 32 rows'
__device__ __forceinline__ int position_at(const PageTable&, const Unit& u, int j, const Sequence&) {
  return (int)u.seq.length - (u.seq.hi - u.seq.lo) + j;
}
__device__ __forceinline__ int least_position(const PageTable& t, const Unit& u, int first, int) { return position_at(t, u, first, u.seq); }
// the last key that new tokens up to j of a unit's rows see
__device__ __forceinline__ int last_seen(const PageTable& t, const Unit& u, int j) { return position_at(t, u, j, u.seq); }

// kChooses: where a workgroup's list of blocks lies
__device__ __forceinline__ int list_of(const PageTable&, char*) { return 0; }

// kSets: sets of 32 rows to a workgroup, which read, and for 8-bit pages convert, K and V once for all of them
template <class E, int D, bool k8, class Table, int kSets>
__global__ __launch_bounds__(64 * kFewWaves, 2) void paged_few_kernel(const PagedParams<E, Table> p) {
  static_assert(kSets == 1 || !kChooses<Table>);
  MOBA_ELEM_TYPES(E)
  using V = std::conditional_t<k8, Bf16, E>;       // type of the second product
  typedef typename V::elem velem;
  typedef typename V::elem4 velem4;
  typedef typename V::elem8 velem8;
  constexpr int kRowBytes = D * (k8 ? 1 : 2), kCols = kRowBytes / 16;
  constexpr int kBlockBytes = kFewKeys * kRowBytes, kStage = 2 * kBlockBytes;
  constexpr int kCopyRows = 64 / kCols, kCopies = kFewKeys / kCopyRows, kSlotCopies = kSlot / kCopyRows;
  constexpr int kSteps = D / 16, kDb = D / 32;     // products of a score block; blocks of 32 output elements
  constexpr int kRedRow = D + 4;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, hh = lane >> 5;
  const auto& shape = p.shape;
  const auto& table = shape.table;
  Unit unit;
  int hkv, item;
  Share share;
  if (!find_unit(shape, p.few, lane, unit, hkv, item, share)) return;
  const Sequence seq = unit.seq;
  if (unit.run == 0 && unit.group == 0 && hkv == 0 && tid == 0) p.runs[item] = {unit.first, unit.runs, unit.groups};
  const int b = unit.row;
  const int count = seq.hi - seq.lo, rows = count * shape.rep, row0 = unit.group * kFewRows * kSets;
  int keys, tiles = unit.tiles;   // kChooses: of the list
  decltype(list_of(table, smem)) list = list_of(table, smem + few_list_at<D, k8>());
  if constexpr (kChooses<Table>) {
    keys = make_list(shape, seq, hkv, row0, min(rows - row0, kFewRows), smem, list);
    tiles = (keys + kFewTile - 1) / kFewTile;
  } else {
    keys = keys_of(shape, seq);
  }
  const int per = (tiles + unit.runs - 1) / unit.runs;   // tiles of a run
  const int key_lo = __builtin_amdgcn_readfirstlane((int)min(seq.begin + (int64_t)unit.run * per * kFewTile, (int64_t)keys));
  const int key_hi = __builtin_amdgcn_readfirstlane((int)min(seq.begin + (int64_t)(unit.run + 1) * per * kFewTile, (int64_t)keys));
  const bool more = kSets > 1 && rows - row0 > kFewRows;   // than one set
  int j[kSets], g[kSets];
  int limit[kSets], first_masked[kSets];   // a row's last visible key (in this run); keys up to here are visible to every row of a set
#pragma unroll
  for (int q = 0; q < kSets; ++q) {
    const int first = min(row0 + q * kFewRows, rows - 1), row = min(first + n, rows - 1);   // (rows past the last repeat it and are not written)
    j[q] = row / shape.rep;
    g[q] = row - j[q] * shape.rep;
    const int position = position_at(table, unit, j[q], share.seq);
    limit[q] = kChooses<Table> ? position : min(position, key_hi - 1);
    first_masked[q] = least_position(table, unit, first / shape.rep, position);
    if constexpr (!kChooses<Table>) first_masked[q] = min(first_masked[q], key_hi - 1);
  }
  const int own_lo = key_lo + wave * kFewKeys;                         // the wave's first key
  const int mine = __builtin_amdgcn_readfirstlane(key_hi > own_lo ? (key_hi - own_lo - 1) / kFewTile + 1 : 0);

  // ---- the wave's copies.  A block is two slots of 16 keys, each inside one page.  Lane i of a copy lands at 16*i, so it picks the
  // global column whose swizzled place that is
  const uint32_t lds_base = lds_addr(smem) + wave * 2 * kStage;
  const uint32_t scale_base = lds_addr(smem) + kFewWaves * 2 * kStage + wave * kScaleBytes;
  uint32_t ld_off[kSlotCopies];
#pragma unroll
  for (int i = 0; i < kSlotCopies; ++i) {
    const int r = i * kCopyRows + lane / kCols;
    ld_off[i] = r * kRowBytes + swizzled<kRowBytes>(r, lane % kCols) * 16;
  }
  const int64_t page_bytes = ((int64_t)shape.Hkv << table.page_log2) * kRowBytes;
  const int64_t head_bytes = ((int64_t)hkv << table.page_log2) * kRowBytes;
  const int page_mask = (1 << table.page_log2) - 1;
  int ids = -1;   // of the wave's slots, 64 at a time
  uint32_t chosen = 0, chosen_now = 0;   // kChooses: the rows that have chosen the slots, and the position of their first keys, of the
  int place = 0, place_now = 0;          // slots of `ids`, and of the batch at hand
  auto fetch_ids = [&](int it0) __attribute__((always_inline)) {
    const int64_t key = own_lo + (int64_t)(it0 + (lane >> 1)) * kFewTile + (lane & 1) * kSlot;
    if constexpr (kChooses<Table>) {
      ids = -1;
      chosen = 0;
      if (key < key_hi) {
        const int page = chosen_page(table, list, (int)key, chosen);
        ids = page_id(table, b, page);
        place = (int)min((int64_t)page << table.page_log2, (int64_t)0x7fff0000) + ((int)key & page_mask);
      }
    } else {
      ids = key < key_hi ? page_id(table, b, key >> table.page_log2) : -1;
    }
    if constexpr (k8) {
      const int64_t at = (int64_t)max(ids, 0) * shape.Hkv + hkv;
      const uint32_t to = scale_base + ((it0 / kBatch) & 1) * (kScaleBytes / 2);
      async_copy4(p.scales[0] + at, to);
      async_copy4(p.scales[1] + at, to + 256);
    }
  };
  auto issue = [&](int it) __attribute__((always_inline)) {
    if (it % kBatch == 0) fetch_ids(it);
    const int key0 = own_lo + it * kFewTile;
    const uint32_t to = lds_base + (it & 1) * kStage;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int slot = 0; slot < 2; ++slot) {
        const int id = __builtin_amdgcn_readlane(ids, (it % kBatch) * 2 + slot);
        const int in_page = (key0 + slot * kSlot) & page_mask;
        // (a slot without a page reads page 0; its keys are masked)
        const char* from = p.pages[half] + head_bytes + (id < 0 ? 0 : id * page_bytes + in_page * kRowBytes);
#pragma unroll
        for (int i = 0; i < kSlotCopies; ++i)
          async_copy16_sv<!kShares<Table>>(from, ld_off[i], to + half * kBlockBytes + (slot * kSlotCopies + i) * 1024);
      }
  };

  // Q^T operands: of step s8, lane (n, hh) holds the 8 elements of row n that its 8 elements of a key meet
  elem8 bq[kSets][kSteps];
#pragma unroll
  for (int q = 0; q < kSets; ++q) {
    const elem* src = p.q + (int64_t)(seq.lo + j[q]) * p.q_tok_stride + (int64_t)(hkv * shape.rep + g[q]) * p.q_head_stride;
#pragma unroll
    for (int s8 = 0; s8 < kSteps; ++s8)
      bq[q][s8] = *reinterpret_cast<const elem8*>(src + (k8 ? 32 * (s8 >> 1) + 16 * hh + 8 * (s8 & 1) : 16 * s8 + 8 * hh));
    // a negative softmax scale: the queries' signs turn, so that the largest product has the largest score
    if (p.scale_log2 < 0.f) {
#pragma unroll
      for (int s8 = 0; s8 < kSteps; ++s8) bq[q][s8] = -bq[q][s8];
    }
  }
  const float scale = fabsf(p.scale_log2);
  if (mine > 0) issue(0);
  if (mine > 1) issue(1);

  // fragment addresses inside stage 0
  constexpr int kKReads = k8 ? kSteps / 2 : kSteps;
  uint32_t koff[kKReads], voff[k8 ? 1 : 2][kDb];
#pragma unroll
  for (int i = 0; i < kKReads; ++i) koff[i] = lds_base + n * kRowBytes + (swizzled<kRowBytes>(n, 2 * i + hh) << 4);
  {
    const int g16 = lane >> 4, l16 = lane & 15;
#pragma unroll
    for (int db = 0; db < kDb; ++db) {
      if constexpr (k8) {
        const int i = l16 >> 1, key = (i < 4 ? i : i + 4) + 4 * hh;
        voff[0][db] = lds_base + kBlockBytes + key * kRowBytes + (swizzled<kRowBytes>(key, 2 * db + (g16 & 1)) << 4) + (l16 & 1) * 8;
      } else {
        const int i0 = l16 >> 2, i1 = l16 & 3, c16 = 4 * db + 2 * (g16 & 1) + (i1 >> 1), sub = (i1 & 1) * 8;
#pragma unroll
        for (int eight = 0; eight < 2; ++eight) {
          const int key = 4 * hh + i0 + 8 * eight;
          voff[eight][db] = lds_base + kBlockBytes + key * kRowBytes + (swizzled<kRowBytes>(key, c16) << 4) + sub;
        }
      }
    }
  }

  f32x16 oacc[kSets][kDb];
  float m_run[kSets], l_run[kSets];
#pragma unroll
  for (int q = 0; q < kSets; ++q) {
    m_run[q] = kNoMax;
    l_run[q] = 0.f;
#pragma unroll
    for (int db = 0; db < kDb; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) oacc[q][db][e] = 0.f;
  }
  uint64_t there = 0;   // the slots of the batch that have a page
  const uint32_t everybody = rows - row0 >= 32 ? ~0u : (1u << (rows - row0)) - 1;

  auto step = [&](int it, auto stage, auto sets) __attribute__((always_inline)) {
    constexpr uint32_t st = stage * kStage;
    constexpr int kHere = sets;
    // (the ids at hand are this batch's: the next batch's are fetched behind its last step but one)
    if (it % kBatch == 0) {
      there = __ballot(ids >= 0);
      chosen_now = chosen;
      place_now = place;
    }
    // this block's copies have landed (the next block's may still be in flight)
    if (it + 1 < mine) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kCopies) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    f32x16 s[kHere];
#pragma unroll
    for (int q = 0; q < kHere; ++q)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[q][e] = 0.f;
    if constexpr (k8) {
      u32x4 raw[kKReads];
#pragma unroll
      for (int i = 0; i < kKReads; ++i) raw[i] = *lds_ptr<const u32x4>(koff[i] + st);
#pragma unroll
      for (int i = 0; i < kKReads; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const elem8 ka = widened(raw[i][2 * half], raw[i][2 * half + 1], E{});
#pragma unroll
          for (int q = 0; q < kHere; ++q) s[q] = mfma32(ka, bq[q][2 * i + half], s[q]);
        }
    } else {
      elem8 ka[kKReads];
#pragma unroll
      for (int i = 0; i < kKReads; ++i) ka[i] = *lds_ptr<const elem8>(koff[i] + st);
#pragma unroll
      for (int i = 0; i < kKReads; ++i)
#pragma unroll
        for (int q = 0; q < kHere; ++q) s[q] = mfma32(ka[i], bq[q][i], s[q]);
    }
    // the V^T fragments travel while the softmax runs
    velem8 va[2][kDb];
    u32x2 vraw[2][kDb];
#pragma unroll
    for (int j2 = 0; j2 < 2; ++j2)
#pragma unroll
      for (int db = 0; db < kDb; ++db) {
        if constexpr (k8) {
          typedef __attribute__((ext_vector_type(2))) int i32x2;
          vraw[j2][db] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                                                       lds_ptr<i32x2>(voff[0][db] + (st + kSlot * j2 * kRowBytes))));
        } else {
          const velem4 x = lds_read_tr<velem4>(voff[0][db] + (st + kSlot * j2 * kRowBytes));
          const velem4 y = lds_read_tr<velem4>(voff[1][db] + (st + kSlot * j2 * kRowBytes));
          va[j2][db] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        }
      }
    const int key0 = own_lo + it * kFewTile;
    // factors of the two slots' scores (not negative: see bq) and probabilities
    float f[kHere][2], vs[2] = {1.f, 1.f};
#pragma unroll
    for (int q = 0; q < kHere; ++q) f[q][0] = f[q][1] = scale;
    if constexpr (k8) {
      const uint32_t at = scale_base + ((it / kBatch) & 1) * (kScaleBytes / 2) + (it % kBatch) * 8;
      const f32x2 k2 = *lds_ptr<const f32x2>(at), v2 = *lds_ptr<const f32x2>(at + 256);
#pragma unroll
      for (int q = 0; q < kHere; ++q) {
        f[q][0] *= k2[0];
        f[q][1] *= k2[1];
      }
      vs[0] = v2[0];
      vs[1] = v2[1];
    }
    const uint32_t has = (uint32_t)(there >> (2 * (it % kBatch))) & 3;
    bool unseen;   // whether there are keys that nobody sees
    if constexpr (kChooses<Table>) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int slot = (it % kBatch) * 2 + half, first = __builtin_amdgcn_readlane(place_now, slot);
        const uint32_t who = (uint32_t)__builtin_amdgcn_readlane((int)chosen_now, slot);
        if (!(has >> half & 1) || (who & everybody) != everybody || first + kSlot - 1 > first_masked[0]) {
          asm volatile("");   // (a branch)
          const bool mine = (has >> half & 1) && (who >> n & 1);
#pragma unroll
          for (int e = 8 * half; e < 8 * half + 8; ++e) {
            s[0][e] *= f[0][half];
            if (!mine || first + 8 * ((e >> 2) & 1) + 4 * hh + (e & 3) > limit[0]) s[0][e] = -INFINITY;
          }
          f[0][half] = 1.f;
        }
      }
      unseen = key0 + kFewKeys > key_hi || has != 3;
    } else {
      unseen = false;
#pragma unroll
      for (int q = 0; q < kHere; ++q)
        if (__builtin_expect(key0 + kFewKeys - 1 > first_masked[q] || has != 3, 0)) {
          asm volatile("");   // (a branch, not sixteen comparisons in every block)
          unseen = true;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            s[q][e] *= f[q][e >> 3];
            if (key0 + 8 * (e >> 2) + 4 * hh + (e & 3) > limit[q] || !(has & (1 << (e >> 3)))) s[q][e] = -INFINITY;
          }
          f[q][0] = f[q][1] = 1.f;
        }
    }
    if (__builtin_expect(unseen, 0)) {
      asm volatile("");
      // their values: whatever lies there
#pragma unroll
      for (int j2 = 0; j2 < 2; ++j2)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (key0 + kSlot * j2 + 8 * (i >> 2) + 4 * hh + (i & 3) >= key_hi || !(has & (1 << j2))) {
#pragma unroll
            for (int db = 0; db < kDb; ++db) {
              if constexpr (k8) vraw[j2][db][i >> 2] &= ~(0xffu << (8 * (i & 3)));
              else va[j2][db][i] = (velem)0.f;
            }
          }
    }
    u32x4 hi[kHere][2], lo[kHere][2];
#pragma unroll
    for (int q = 0; q < kHere; ++q) {
      float mx[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        mx[half] = s[q][8 * half];
#pragma unroll
        for (int e = 1; e < 8; ++e) mx[half] = fmaxf(mx[half], s[q][8 * half + e]);
      }
      mx[0] = max_xhalf(fmaxf(mx[0] * f[q][0], mx[1] * f[q][1]));
      if (__any(mx[0] > m_run[q] + kMaxLag)) {  // rare once the maximum has settled
        const float m_new = mx[0] > m_run[q] + kMaxLag ? mx[0] : m_run[q];
        const float alpha = fast_exp2(m_run[q] - m_new);
        m_run[q] = m_new;
        l_run[q] *= alpha;
#pragma unroll
        for (int db = 0; db < kDb; ++db)
#pragma unroll
          for (int e = 0; e < 16; ++e) oacc[q][db][e] *= alpha;
      }
      const float ref = m_run[q] - ProbShift<V>::value;
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        float p0 = fast_exp2(fmaf(s[q][e], f[q][e >> 3], -ref)), p1 = fast_exp2(fmaf(s[q][e + 1], f[q][e >> 3], -ref));
        l_run[q] += p0;
        l_run[q] += p1;
        if constexpr (k8) {
          p0 *= vs[e >> 3];
          p1 *= vs[e >> 3];
        }
        uint32_t h, l;
        in_two<V>(p0, p1, h, l);
        hi[q][e >> 3][(e & 7) >> 1] = h;
        lo[q][e >> 3][(e & 7) >> 1] = l;
      }
    }
    if constexpr (k8) {
#pragma unroll
      for (int j2 = 0; j2 < 2; ++j2)
#pragma unroll
        for (int db = 0; db < kDb; ++db) va[j2][db] = widened(vraw[j2][db][0], vraw[j2][db][1], Bf16{});
    }
#pragma unroll
    for (int q = 0; q < kHere; ++q) {
#pragma unroll
      for (int j2 = 0; j2 < 2; ++j2)
#pragma unroll
        for (int db = 0; db < kDb; ++db) oacc[q][db] = mfma32(va[j2][db], __builtin_bit_cast(velem8, hi[q][j2]), oacc[q][db]);
#pragma unroll
      for (int j2 = 0; j2 < 2; ++j2)
#pragma unroll
        for (int db = 0; db < kDb; ++db) oacc[q][db] = mfma32(va[j2][db], __builtin_bit_cast(velem8, lo[q][j2]), oacc[q][db]);
    }
    if (it + 2 < mine) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every fragment of this stage is in registers
      issue(it + 2);
    }
  };
  // (the stage is a constant of each copy of the body, and part of its LDS instructions)
  auto all_steps = [&](auto sets) __attribute__((always_inline)) {
    for (int it = 0; it < mine; it += 2) {
      step(it, std::integral_constant<int, 0>{}, sets);
      if (it + 1 < mine) step(it + 1, std::integral_constant<int, 1>{}, sets);
    }
  };
  if constexpr (kSets > 1) {
    if (more) all_steps(std::integral_constant<int, kSets>{});
    else all_steps(std::integral_constant<int, 1>{});
  } else {
    all_steps(std::integral_constant<int, 1>{});
  }
#pragma unroll
  for (int q = 0; q < kSets; ++q) {
    if (__builtin_expect(__any(any_not_finite(oacc[q])), 0))  // (never for values of ordinary size)
      one_by_one<E, V, D, k8, k8>(p, hkv, own_lo, kFewTile, key_hi, [&](int key, bool& sees) __attribute__((always_inline)) {
        if constexpr (kChooses<Table>) {
          uint32_t who;
          const int page = chosen_page(table, list, key, who);
          sees = (who >> n & 1) && ((int64_t)page << table.page_log2) + (key & page_mask) <= limit[q];
          return page_id(table, b, page);
        } else {
          sees = key <= limit[q];
          return page_id(table, b, key >> table.page_log2);
        }
      }, scale, bq[q], oacc[q], m_run[q], l_run[q]);
    l_run[q] = sum_xhalf(l_run[q]);
  }

  // ---- the waves meet in LDS.  Element e of lane (n, hh) is O[row n][32*db + 8*(e/4) + 4*hh + e%4].
  float* red = reinterpret_cast<float*>(smem);
  float* red_m = red + kFewWaves * 32 * kRedRow;
  float* red_l = red_m + kFewWaves * 32;
#pragma unroll
  for (int q = 0; q < kSets; ++q) {
    const int first = row0 + q * kFewRows, rows_here = min(kFewRows, rows - first);
    if (q && rows_here <= 0) break;
    __syncthreads();  // every wave has read its last fragments, or the former set's rows
    if (n < rows_here) {
#pragma unroll
      for (int db = 0; db < kDb; ++db)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4)
          *reinterpret_cast<f32x4*>(red + (wave * 32 + n) * kRedRow + 32 * db + 8 * g4 + 4 * hh) =
              f32x4{oacc[q][db][4 * g4], oacc[q][db][4 * g4 + 1], oacc[q][db][4 * g4 + 2], oacc[q][db][4 * g4 + 3]};
      if (hh == 0) {
        red_m[wave * 32 + n] = m_run[q];
        red_l[wave * 32 + n] = l_run[q];
      }
    }
    __syncthreads();
    for (int i = tid; i < rows_here * (D / 4); i += 64 * kFewWaves) {
      const int rr = i / (D / 4), d = (i % (D / 4)) * 4;
      float mm = red_m[rr];
#pragma unroll
      for (int w = 1; w < kFewWaves; ++w) mm = fmaxf(mm, red_m[w * 32 + rr]);
      float ll = 0.f;
      f32x4 oo = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) {
        const float a = fast_exp2(red_m[w * 32 + rr] - mm);
        ll += red_l[w * 32 + rr] * a;
        const f32x4 x = *reinterpret_cast<const f32x4*>(red + (w * 32 + rr) * kRedRow + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) oo[e] += x[e] * a;
      }
      const float inv = ll == 0.f ? 0.f : 1.f / ll;   // (a row may see no key of its run, or none at all)
      if (!kShares<Table> && unit.runs == 1) {
        const int jj = (first + rr) / shape.rep, gg = first + rr - jj * shape.rep;
        const int64_t orow = (int64_t)(seq.lo + jj) * shape.H + hkv * shape.rep + gg;
        *reinterpret_cast<u32x2*>(p.out + orow * D + d) = u32x2{pack2<E>(oo[0] * inv, oo[1] * inv), pack2<E>(oo[2] * inv, oo[3] * inv)};
      } else {
        const int64_t number = blockIdx.x + (int64_t)first_unit(table) * shape.Hkv, prow = (number * kSets + q) * kFewRows + rr;
        *reinterpret_cast<f32x4*>(p.few_o + prow * D + d) = f32x4{oo[0] * inv, oo[1] * inv, oo[2] * inv, oo[3] * inv};
        if (d == 0) p.few_lse[prow] = ll == 0.f ? -INFINITY : mm - ProbShift<V>::value + fast_log2(ll);
      }
    }
  }
}

// ---- many rows: bound by the products and, beside them, by the vector instructions of the softmax and of the 8-bit elements.  A
// workgroup takes 32 rows to a wave; tiles of 64 keys are brought into LDS once for all of them, in rings of three K and two V
// tiles, one barrier a tile.  16-bit tiles are copied global -> LDS, four waves to a workgroup and two workgroups to a compute unit, so
// that one's lookups and barriers run under the other's products.  8-bit tiles come through registers, where they become 16-bit
// elements: eight waves share that work where heads have 128 elements, one workgroup to a compute unit (2048 tokens against 34816
// keys, 32 and 8 heads, the whole call: 1067 us, with four waves 1145; 16-bit pages: 1129 with eight, 1111 with four, and 2048 tokens
// without a cache 77 and 70).  Priority for the products gives 4 % with four waves and takes 2 % with eight.
constexpr int kManyKeys = 64;
template <int D, bool k8> constexpr int kManyWaves = D == 128 && k8 ? 8 : 4;

// A tile lies in LDS in the order in which its fragments are read, so that a read's address is a constant of the lane and a
// constant of the instruction, and no two lanes meet in a bank:
//   K  for each block of 32 keys and step of 16 elements the 64 lanes' 16 bytes, lane (n, hh): elements 8hh .. of key n
//   V  for each 16 elements and 4 keys (16 such in a row) 128 bytes, the keys one behind the other, which a transposing read of
//      16 lanes takes; of odd 16 elements every two of these have changed places, so that the even and the odd that are read
//      together lie in different banks
// (Rows instead, their columns swizzled by exclusive or, took 13 address registers more; rows with 32 bytes between them, three times the
// bank conflicts.)
template <int D>
constexpr int many_lds_bytes() { return 5 * kManyKeys * D * 2; }

// Elements of a probability: one, rounded, of the queries' own precision; where queries are fp16 and the products bf16, two.
template <class E, class V> struct ProbParts { static constexpr int value = 2; };
template <class E> struct ProbParts<E, E> { static constexpr int value = 1; };

template <class E, int D, bool k8, class Table>
__global__ __launch_bounds__(64 * (kManyWaves<D, k8>), 2) void paged_many_kernel(const PagedParams<E, Table> p) {
  MOBA_ELEM_TYPES(E)
  using V = std::conditional_t<k8, Bf16, E>;
  typedef typename V::elem velem;
  typedef typename V::elem4 velem4;
  typedef typename V::elem8 velem8;
  constexpr int kWaves = kManyWaves<D, k8>, kRows = 32 * kWaves;
  constexpr int kParts = ProbParts<E, V>::value;
  constexpr int kTileBytes = kManyKeys * D * 2;
  constexpr int kRow = D * (k8 ? 1 : 2);                                   // in the pages
  constexpr int kPieces = kManyKeys * kRow / 16 / (64 * kWaves);       // 16-byte pieces of a tile of K (or V) of a thread
  constexpr int kSteps = D / 16, kDb = D / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, hh = lane >> 5;
  const auto& shape = p.shape;
  const auto& table = shape.table;
  Unit unit;
  int hkv, item;
  Share share;
  if (!find_unit(shape, p.many, lane, unit, hkv, item, share)) return;
  const Sequence seq = unit.seq;
  const int keys = keys_of(shape, seq);
  if (unit.run == 0 && unit.group == 0 && hkv == 0 && tid == 0) p.runs[item] = {unit.first, unit.runs, unit.groups};
  const int b = unit.row;
  // (the group with the most keys first)
  const int count = seq.hi - seq.lo, rows = count * shape.rep, row0 = (unit.groups - 1 - unit.group) * kRows;
  const int per = (unit.tiles + unit.runs - 1) / unit.runs;
  const int last_row = min(row0 + kRows, rows) - 1;
  const int seen = max(min(keys, last_seen(table, unit, last_row / shape.rep) + 1), seq.begin);   // the end of what the group's last row sees
  const int key_lo = (int)min(seq.begin + (int64_t)unit.run * per * kManyKeys, (int64_t)seen);
  const int key_hi = (int)min(seq.begin + (int64_t)(unit.run + 1) * per * kManyKeys, (int64_t)seen);
  const int wave_row = row0 + 32 * wave;
  const int row = min(wave_row + n, rows - 1);
  const int j = row / shape.rep, g = row - j * shape.rep;
  const int position = position_at(table, unit, j, share.seq);
  const int limit = min(position, key_hi - 1);
  const int first_masked = min(least_position(table, unit, min(wave_row, rows - 1) / shape.rep, position), key_hi - 1);
  const int tiles = (key_hi - key_lo + kManyKeys - 1) / kManyKeys;
  const bool works = wave_row < rows;

  // ---- copies.  A run begins at a multiple of 64 keys, so where in its page a piece lies is a constant of the thread and, in
  // pages of more than 64 tokens, the tile's place.  Keys behind the run's last are masked, and read its page again; where the table
  // names no page, page 0 is read.
  //   8-bit: piece c of a thread is 16 elements, `col`, of the key key_of(c), of K and of V
  //   16-bit: piece c of a wave is the 1 KiB copy 4c + wave of the tile; of K step (4c + wave) % kSteps of a block of 32 keys, of V
  //   the half wave % 2 of the keys and 16 elements
  constexpr int kKeysAtOnce = k8 ? 64 * kWaves * 16 / kRow : 32;
  const uint32_t page_bytes = (uint32_t)shape.Hkv * kRow << table.page_log2;
  const int64_t head_bytes = ((int64_t)hkv << table.page_log2) * kRow;
  const int page_mask = (1 << table.page_log2) - 1;
  const int32_t* const page_row = table.pages + b * table.stride;
  const uint32_t lds = lds_addr(smem);
  constexpr int kLookups = k8 ? kPieces : 2;
  const int col = k8 ? tid / kKeysAtOnce : 0;
  auto key_of = [&](int c) { return (k8 ? tid % kKeysAtOnce : n) + c * kKeysAtOnce; };
  const int v_key = 32 * (wave & 1) + 4 * ((lane >> 3) ^ ((wave >> 1) & 1)) + ((lane & 7) >> 1);   // 16-bit: of V
  uint32_t in_page[kLookups];
#pragma unroll
  for (int c = 0; c < kLookups; ++c) in_page[c] = (key_of(c) & page_mask) * kRow + (k8 ? col : hh) * 16;
  const uint32_t v_in_page = (v_key & page_mask) * kRow + (lane & 1) * 16;
  auto look_up = [&](int key) __attribute__((always_inline)) {   // the page of a key of the run, -1 where there is none
    const int id = page_row[(uint32_t)min(key, key_hi - 1) >> table.page_log2];
    return (uint32_t)id < (uint32_t)table.num_pages ? id : -1;
  };
  int ids[kLookups], v_ids[k8 ? kPieces : 1], v_id = 0;   // of the tiles of which K and V are fetched next (v_id: 16-bit, V of K's tile)
  // Of the tile at hand, the next and the one behind it: the place of its K, the slots of 16 keys that have a page, and in lane i K's
  // scale of slot i % 4.
  uint32_t place[3], there[3] = {};
  float k_scale[3] = {};
  uint32_t v_place[2];               // V of the tile at hand and of the next
  int slot_id = -1, slot_id2 = -1;   // lane i: the page of slot i % 4 of the tile whose K has been asked for, and of the next
  float slot_scale = 0.f;
  auto fetch_ids = [&](int t) __attribute__((always_inline)) {
    const int key0 = key_lo + t * kManyKeys;
#pragma unroll
    for (int c = 0; c < kLookups; ++c) ids[c] = max(look_up(key0 + key_of(c)), 0);
    if constexpr (!k8) v_id = max(look_up(key0 + v_key), 0);
    const int key = key0 + (lane & 3) * kSlot, id = look_up(key);
    slot_id2 = key < key_hi ? id : -1;
  };
  u32x4 raw[2][k8 ? kPieces : 1];
  float raw_scale[k8 ? kPieces : 1];   // V's of the pieces
  auto in_tile = [&](int t) { return head_bytes + (int64_t)((key_lo + t * kManyKeys) & page_mask & -kManyKeys) * kRow; };
  auto fetch_k = [&](int t, uint32_t to) __attribute__((always_inline)) {
    const char* const from = p.pages[0] + in_tile(t);
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      if constexpr (k8) {
        raw[0][c] = *reinterpret_cast<const u32x4*>(from + ((uint64_t)(uint32_t)ids[c] * page_bytes + in_page[c]));
      } else {
        const int copy = c * kWaves + wave, blk = c * kWaves / kSteps;
        async_copy16(from + ((uint64_t)(uint32_t)ids[blk] * page_bytes + in_page[blk]) + copy % kSteps * 32, lds + to + copy * 1024);
      }
    }
    slot_id = slot_id2;
    if constexpr (k8) slot_scale = p.scales[0][(uint32_t)max(slot_id, 0) * (uint64_t)(uint32_t)shape.Hkv + hkv];
  };
  auto fetch_v = [&](int t, uint32_t to) __attribute__((always_inline)) {
    const char* const from = p.pages[1] + in_tile(t);
    if constexpr (k8) {
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        raw[1][c] = *reinterpret_cast<const u32x4*>(from + ((uint64_t)(uint32_t)v_ids[c] * page_bytes + in_page[c]));
        raw_scale[c] = p.scales[1][(uint32_t)v_ids[c] * (uint64_t)(uint32_t)shape.Hkv + hkv];
      }
    } else {
      const char* const row = from + ((uint64_t)(uint32_t)v_ids[0] * page_bytes + v_in_page);
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        const int copy = c * kWaves + wave;
        async_copy16(row + (copy >> 1) * 32, lds + to + copy * 1024);
      }
    }
  };
  // V's rows of keys that nobody sees hold whatever lies there, and become zeros
  auto unseen = [&](int t, uint32_t has) { return key_lo + (t + 1) * kManyKeys > key_hi || has != 15; };
  auto key_unseen = [&](int t, uint32_t has, int key) {
    return key_lo + t * kManyKeys + key >= key_hi || !((has >> (key >> 4)) & 1);
  };
  // 8-bit: what the fetches have brought goes to its place
  auto store_k = [&](uint32_t to) __attribute__((always_inline)) {
    if constexpr (k8) {
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        const int key = key_of(c);
        const uint32_t at = lds + to + (((key >> 5) * kSteps + col) * 64 + (key & 31)) * 16;
        const u32x4 w = raw[0][c];
        *lds_ptr<elem8>(at) = widened(w[0], w[1], E{});
        *lds_ptr<elem8>(at + 512) = widened(w[2], w[3], E{});
      }
    }
  };
  auto store_v = [&](int t, uint32_t to, uint32_t has) __attribute__((always_inline)) {
    if constexpr (k8) {
      bool odd = false;   // (no scale of paged_append's)
#pragma unroll
      for (int c = 0; c < kPieces; ++c) odd |= !power_of_two(raw_scale[c]);
      auto put = [&](auto plain) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
          const int key = key_of(c);
          const uint32_t at = lds + to + (col * 16 + ((key >> 2) ^ (col & 1))) * 128 + (key & 3) * 32;
          u32x4 w = raw[1][c];
          bf16x8 v0, v1;
          if constexpr (plain) {
            v0 = widened(w[0], w[1], Bf16{}, raw_scale[c]);
            v1 = widened(w[2], w[3], Bf16{}, raw_scale[c]);
          } else {
            const bool none = key_unseen(t, has, key);
            if (none) w = u32x4{0, 0, 0, 0};
            const float by = none ? 1.f : raw_scale[c];
            v0 = widened_by(w[0], w[1], by);
            v1 = widened_by(w[2], w[3], by);
          }
          *lds_ptr<bf16x8>(at) = v0;
          *lds_ptr<bf16x8>(at + 16) = v1;
        }
      };
      if (__builtin_expect(unseen(t, has) || __any(odd), 0)) put(std::false_type{});
      else put(std::true_type{});
    }
  };
  // 16-bit: the thread's own copies have landed
  auto landed = [&](int t, uint32_t to, uint32_t has) __attribute__((always_inline)) {
    if constexpr (!k8) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (__builtin_expect(unseen(t, has), 0)) {
        asm volatile("");
        if (key_unseen(t, has, v_key)) {
#pragma unroll
          for (int c = 0; c < kPieces; ++c)
            *lds_ptr<u32x4>(lds + to + c * 64 * kWaves * 16 + tid * 16) = u32x4{0, 0, 0, 0};
        }
      }
    }
  };

  elem8 bq[kSteps];
  {
    const elem* src = p.q + (int64_t)(seq.lo + j) * p.q_tok_stride + (int64_t)(hkv * shape.rep + g) * p.q_head_stride + 8 * hh;
#pragma unroll
    for (int s8 = 0; s8 < kSteps; ++s8) bq[s8] = *reinterpret_cast<const elem8*>(src + 16 * s8);
    // a negative softmax scale: the queries' signs turn, so that the largest product has the largest score
    if (p.scale_log2 < 0.f) {
#pragma unroll
      for (int s8 = 0; s8 < kSteps; ++s8) bq[s8] = -bq[s8];
    }
  }
  const float scale = fabsf(p.scale_log2);
  const uint32_t k_lane = lds + lane * 16;
  const uint32_t v_lane = lds + ((lane >> 4) & 1) * 2048 + (hh ^ ((lane >> 4) & 1)) * 128 + (lane & 15) * 8;
  f32x16 oacc[kDb];
  float m_run = kNoMax, l_run = 0.f;

  // At the beginning of tile t's work K of tile t + 2 and V of tile t + 1 go to LDS, and are complete long before the barrier at its end:
  // 8-bit tiles from registers, which the fetches fill again with the tiles behind; 16-bit ones from memory.
  auto bring_k = [&](int t, int at) __attribute__((always_inline)) {
    if constexpr (!k8) fetch_k(t, place[at]);
    there[at] = (uint32_t)__ballot(slot_id >= 0) & 15;
    k_scale[at] = slot_scale;
    store_k(place[at]);
    if constexpr (k8) fetch_k(t + 1, 0);
  };
  auto bring_v = [&](int t, int at) __attribute__((always_inline)) {
    if constexpr (!k8) fetch_v(t, v_place[at]);
    store_v(t, v_place[at], there[at]);
    if constexpr (k8) fetch_v(t + 1, 0);
  };
  auto next_ids = [&](int t) __attribute__((always_inline)) {
    if constexpr (k8) {
#pragma unroll
      for (int c = 0; c < kPieces; ++c) v_ids[c] = ids[c];
    } else {
      v_ids[0] = v_id;
    }
    fetch_ids(t);
  };
  auto barrier = [&]() __attribute__((always_inline)) {
    // (the wave's LDS instructions are done; loads to registers may be on their way)
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };

  auto k_frag = [&](uint32_t st, int blk, int i) __attribute__((always_inline)) {
    return *lds_ptr<const elem8>(k_lane + st + (blk * kSteps + i) * 1024);
  };
  auto v_frag = [&](uint32_t st, int blk, int j2, int db) __attribute__((always_inline)) {
    const uint32_t at = v_lane + st + (db * 4096 + (8 * blk + 4 * j2) * 128);   // keys 4hh .., and 8 + 4hh .. of 16
    const velem4 x = lds_read_tr<velem4>(at), y = lds_read_tr<velem4>(at + 256);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // masks what a row does not see of a block's scores; f: the factors of their halves (of 16 keys)
  auto mask = [&](int key0, int blk, int tile, f32x16& s, float (&f)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int half = 0; half < 2; ++half) f[half] = k8 ? lane_value(k_scale[tile], 2 * blk + half) * scale : scale;
    const uint32_t has = (there[tile] >> (2 * blk)) & 3;
    if (__builtin_expect(key0 + 32 * blk + 31 > first_masked || has != 3, 0)) {
      asm volatile("");   // (a branch, not sixteen comparisons in every block)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] *= f[e >> 3];
        if (key0 + 32 * blk + 8 * (e >> 2) + 4 * hh + (e & 3) > limit || !(has & (1 << (e >> 3)))) s[e] = -INFINITY;
      }
      f[0] = f[1] = 1.f;
    }
  };
  auto largest = [&](const f32x16& s, const float (&f)[2]) __attribute__((always_inline)) {   // of a row's scores
    float mx[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      mx[half] = s[8 * half];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx[half] = fmaxf(mx[half], s[8 * half + e]);
    }
    return max_xhalf(fmaxf(mx[0] * f[0], mx[1] * f[1]));
  };
  velem8 hi[2], lo[2];   // a block's probabilities
  auto exponentials = [&](f32x16& s, const float (&f)[2], int from, int to) __attribute__((always_inline)) {
    const float ref = m_run - ProbShift<V>::value;
#pragma unroll
    for (int e = from; e < to; ++e) {
      s[e] = fast_exp2(fmaf(s[e], f[e >> 3], -ref));
      l_run += s[e];
      asm volatile("" : "+v"(s[e]), "+v"(l_run));
    }
  };
  auto pack = [&](const f32x16& s, int half) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const velem h = (velem)s[8 * half + e];
      hi[half][e] = h;
      if constexpr (kParts == 2) lo[half][e] = (velem)(s[8 * half + e] - (float)h);
    }
  };

  // All keys of the run, in blocks of 32, by hand in slots of one matrix instruction and the vector instructions beside it: the
  // scores of the next block under the second half of this one's exponentials, this one's probabilities times V under
  // the first half of the next one's.  kFixed: relative to the maximum of the first block (false where a row has none);
  // otherwise with a running maximum.
  auto all_keys = [&](auto fixed) __attribute__((always_inline)) {
    constexpr bool kFixed = fixed;
#pragma unroll
    for (int i = 0; i < 3; ++i) place[i] = i * kTileBytes;
#pragma unroll
    for (int i = 0; i < 2; ++i) v_place[i] = (3 + i) * kTileBytes;
    fetch_ids(0);
    if constexpr (k8) {
      fetch_k(0, 0);
      next_ids(1);
      fetch_v(0, 0);
    }
    bring_k(0, 0);
    next_ids(k8 ? 2 : 1);
    bring_v(0, 0);
    bring_k(1, 1);
    next_ids(k8 ? 3 : 2);
    landed(0, v_place[0], there[0]);   // (16-bit: K of tile 1 among what is waited for)
    barrier();
#pragma unroll
    for (int db = 0; db < kDb; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) oacc[db][e] = 0.f;
    l_run = 0.f;
    f32x16 s0, s1;
    float f0[2], f1[2];
    elem8 ahead[kSteps / 2];   // the first K fragments of the next scores
#pragma unroll
    for (int e = 0; e < 16; ++e) s0[e] = 0.f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) s0 = mfma32(k_frag(0, 0, i), bq[i], s0);
#pragma unroll
    for (int i = 0; i < kSteps / 2; ++i) ahead[i] = k_frag(0, 1, i);
    mask(key_lo, 0, 0, s0, f0);
    const float m = largest(s0, f0);
    const bool found = m > kNoMax;
    m_run = found ? m : kFixed ? 0.f : kNoMax;
    exponentials(s0, f0, 0, 8);
    pack(s0, 0);

    // sc: the scores of block blk of the tile at hand, of which the first half is in hi[0]; sn takes those of the next block, in
    // tile `next` of the three; then, K fragments of block `blk` of tile 1 are next
    auto step = [&](f32x16& sc, float (&fc)[2], f32x16& sn, float (&fn)[2], auto blk, auto has_next, int key0, bool more)
        __attribute__((always_inline)) {
      constexpr int kNext = blk;   // tile of the next block
      velem8 va[2][kDb];
      elem8 ka[kSteps];
      if constexpr (has_next) {
#pragma unroll
        for (int i = 0; i < kSteps / 2; ++i) ka[i] = ahead[i];
#pragma unroll
        for (int e = 0; e < 16; ++e) sn[e] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if constexpr (has_next) {
          if (i + kSteps / 2 < kSteps) ka[i + kSteps / 2] = k_frag(place[kNext], 1 - blk, i + kSteps / 2);
          sn = mfma32(ka[i], bq[i], sn);
        }
        exponentials(sc, fc, 8 + 8 * i / kSteps, 8 + 8 * (i + 1) / kSteps);
        if (i >= kSteps / 2) {
#pragma unroll
          for (int db = (i - kSteps / 2) * kDb * 2 / kSteps; db < (i - kSteps / 2 + 1) * kDb * 2 / kSteps; ++db)
            va[0][db] = v_frag(v_place[0], blk, 0, db);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      pack(sc, 1);
      if constexpr (has_next) mask(key0 + kNext * kManyKeys, 1 - blk, kNext, sn, fn);
#pragma unroll
      for (int k = 0; k < 2 * kDb; ++k) {
        if (k < kDb) va[1][k] = v_frag(v_place[0], blk, 1, k);
        if constexpr (has_next) {
          if (k >= kDb && more) {
#pragma unroll
            for (int i = (k - kDb) * kSteps / (2 * kDb); i < (k - kDb + 1) * kSteps / (2 * kDb); ++i) ahead[i] = k_frag(place[1], blk, i);
          }
        }
        oacc[k % kDb] = mfma32(va[k / kDb][k % kDb], hi[k / kDb], oacc[k % kDb]);
        if constexpr (kParts == 2) oacc[k % kDb] = mfma32(va[k / kDb][k % kDb], lo[k / kDb], oacc[k % kDb]);
        if constexpr (has_next && kFixed) {   // (the first slot is left to the last score product's result)
          const int from = k == 0 ? 0 : 8 * (k - 1) / (2 * kDb - 1), to = k == 0 ? 0 : 8 * k / (2 * kDb - 1);
          exponentials(sn, fn, from, to);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (has_next && !kFixed) {
        const float mm = largest(sn, fn);
        if (__any(mm > m_run + kMaxLag)) {
          const float m_new = mm > m_run + kMaxLag ? mm : m_run;
          const float alpha = fast_exp2(m_run - m_new);
          m_run = m_new;
          l_run *= alpha;
#pragma unroll
          for (int db = 0; db < kDb; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) oacc[db][e] *= alpha;
        }
        exponentials(sn, fn, 0, 8);
      }
      if constexpr (has_next) pack(sn, 0);
    };
    constexpr std::integral_constant<int, 0> k0;
    constexpr std::integral_constant<int, 1> k1;
    int key0 = key_lo;
    for (int t = 0; t + 1 < tiles; ++t, key0 += kManyKeys) {
      const bool two_more = t + 2 < tiles;
      if (two_more) bring_k(t + 2, 2);
      bring_v(t + 1, 1);
      next_ids(t + (k8 ? 4 : 3));
      if (works) {
        if constexpr (kWaves == 4) __builtin_amdgcn_s_setprio(1);
        step(s0, f0, s1, f1, k0, std::true_type{}, key0, true);
        step(s1, f1, s0, f0, k1, std::true_type{}, key0, true);
        if constexpr (kWaves == 4) __builtin_amdgcn_s_setprio(0);
      }
      landed(t + 1, v_place[1], there[1]);
      barrier();   // what was brought is complete, and nobody reads tile t any more
      const uint32_t free = place[0];
      place[0] = place[1]; place[1] = place[2]; place[2] = free;
      const uint32_t v_free = v_place[0];
      v_place[0] = v_place[1]; v_place[1] = v_free;
      there[0] = there[1]; there[1] = there[2];
      k_scale[0] = k_scale[1]; k_scale[1] = k_scale[2];
    }
    step(s0, f0, s1, f1, k0, std::true_type{}, key0, false);
    step(s1, f1, s0, f0, k1, std::false_type{}, key0, false);
    return found;
  };
  if (tiles > 0) {
    constexpr bool kFixed = std::is_same_v<V, Bf16>;
    bool again = !kFixed;
    if constexpr (kFixed) {
      const bool found = all_keys(std::true_type{});
      const float sum = sum_xhalf(l_run);
      // (a row whose first keys have no page has no reference)
      const bool bad = wave_row + n < rows && (float_bits(sum) >= float_bits(0x1p96f) || any_not_finite(oacc) || (!found && limit >= key_lo));
      __syncthreads();   // (everybody has read the last tile)
      volatile int* const flags = reinterpret_cast<volatile int*>(smem);
      const bool any_bad = __any(bad);
      if (lane == 0) flags[wave] = any_bad;
      __syncthreads();
      int some = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) some |= flags[w];
      again = __builtin_amdgcn_readfirstlane(some) != 0;
      __syncthreads();   // (everybody has read the flags)
    }
    if (__builtin_expect(again, 0)) all_keys(std::false_type{});
  } else {
#pragma unroll
    for (int db = 0; db < kDb; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) oacc[db][e] = 0.f;
  }
  if (!works) return;   // (no barrier follows)
  if (__builtin_expect(__any(any_not_finite(oacc)), 0))
    one_by_one<E, V, D, k8, false>(p, hkv, key_lo, 32, key_hi, [&](int key, bool& sees) __attribute__((always_inline)) {
      sees = key <= limit;
      return page_id(table, b, key >> table.page_log2);
    }, scale, bq, oacc, m_run, l_run);
  l_run = sum_xhalf(l_run);
  if (wave_row + n >= rows) return;
  const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
  if (!kShares<Table> && unit.runs == 1) {
    elem* to = p.out + ((int64_t)(seq.lo + j) * shape.H + hkv * shape.rep + g) * D + 4 * hh;
#pragma unroll
    for (int i = 0; i < 4 * kDb; ++i) {
      const f32x16& o = oacc[i >> 2];
      const int e = 4 * (i & 3);
      *reinterpret_cast<u32x2*>(to + 8 * i) = u32x2{pack2<E>(o[e] * inv, o[e + 1] * inv), pack2<E>(o[e + 2] * inv, o[e + 3] * inv)};
    }
  } else {
    const int64_t prow = (int64_t)blockIdx.x * kRows + 32 * wave + n;
#pragma unroll
    for (int i = 0; i < 4 * kDb; ++i) {
      const f32x16& o = oacc[i >> 2];
      const int e = 4 * (i & 3);
      *reinterpret_cast<f32x4*>(p.many_o + prow * D + 8 * i + 4 * hh) = f32x4{o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv};
    }
    if (hh == 0) p.many_lse[prow] = l_run == 0.f ? -INFINITY : m_run - ProbShift<V>::value + fast_log2(l_run);
  }
}

// Where the parts of a row lie: `runs` of them, row `first` + i * `step` of part_o and part_lse each
struct Parts {
  const float *o, *lse;
  int runs;
  int64_t first, step;
};

// The units that have left parts of a token's rows: their sequences' numbers, which of their new tokens it is, and how many of those
// there are; keys: whether there is any
struct Side {
  int unit, token, count;
  bool keys;
};
// of token t, found with the whole wave
template <class Table>
__device__ __forceinline__ void sides_of(const Shape<Table>& shape, int t, int lane, Side (&side)[1]) {
  Sequence seq = {};
  const int b = last_up_to(shape.table, t, lane, seq, [](int, int lo) { return (int64_t)lo; });
  side[0] = {b, t - seq.lo, seq.hi - seq.lo, b >= 0 && t < seq.hi && keys_of(shape, seq) > 0};
}

// What the merge has found of a token
template <class E, class Table>
struct MergeToken {
  static constexpr int kSides = kShares<Table> ? 2 : 1;
  Side side[kSides];
  Runs r[kSides];
  bool is_many[kSides];
  __device__ __forceinline__ MergeToken(const PagedParams<E, Table>& p, int t, int lane) {
    sides_of(p.shape, t, lane, side);
#pragma unroll
    for (int s = 0; s < kSides; ++s) {
      r[s] = {0, 0, 0};
      is_many[s] = side[s].count * p.shape.rep > p.many.rows_over && p.many.most > 0;
      if (side[s].keys) {   // (its units have left their numbers)
        const Runs x = p.runs[side[s].unit];
        r[s] = {__builtin_amdgcn_readfirstlane(x.first), __builtin_amdgcn_readfirstlane(x.runs), __builtin_amdgcn_readfirstlane(x.groups)};
      }
    }
  }
  __device__ __forceinline__ bool done() const { return kSides == 1 && r[0].runs == 1; }   // (the only run's unit has written the rows)
  // of query head g of key/value head hkv (group_rows is a power of two)
  __device__ __forceinline__ Parts parts(const PagedParams<E, Table>& p, int hkv, int g, int s) const {
    const Cut& cut = is_many[s] ? p.many : p.few;
    const int row = side[s].token * p.shape.rep + g;
    int group = row >> (31 - __builtin_clz(cut.group_rows));
    const int rr = row & (cut.group_rows - 1);
    if (is_many[s]) group = r[s].groups - 1 - group;
    // (numbers that no unit has left, where the row ranges are none)
    const bool none = r[s].first < 0 || r[s].runs < 0 || r[s].groups < 1 || r[s].first + (int64_t)r[s].runs * r[s].groups > cut.parts ||
                      group < 0 || group >= r[s].groups;
    return {is_many[s] ? p.many_o : p.few_o, is_many[s] ? p.many_lse : p.few_lse, none ? 0 : r[s].runs,
            (((int64_t)r[s].first + group) * p.shape.Hkv + hkv) * cut.group_rows + rr, (int64_t)r[s].groups * p.shape.Hkv * cut.group_rows};
  }
};

// `heads` heads of a token, one after the other, for kShare waves, a lane for D / 64 elements.  Four waves (few tokens, which may
// have many runs) take a quarter of the runs each, their sums meet in LDS; one wave needs neither.  Rows of one run are there already.
// Bound by its chain of reads (sequence, its number of runs, log-sum-exps and rows): 4.7 us for one token.
template <class E, int D, int kShare, class Table>
__global__ __launch_bounds__(256) void paged_merge_kernel(const PagedParams<E, Table> p, int heads) {
  typedef typename E::elem elem;
  constexpr int kPer = D / 64;
  typedef float fvec __attribute__((ext_vector_type(kPer)));
  __shared__ float red[4][D];
  __shared__ float red_l[4];
  const int lane = threadIdx.x & 63, wave_in_group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = kShare == 4 ? wave_in_group : 0;
  const auto& shape = p.shape;
  const auto& table = shape.table;
  const int per_token = (shape.H + heads - 1) / heads;
  const int item = kShare == 4 ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave_in_group;
  const int t = item / per_token, h0 = (item - t * per_token) * heads;
  if (t >= table.T) return;
  constexpr int kSides = kShares<Table> ? 2 : 1;
  const MergeToken<E, Table> token(p, t, lane);
  if (token.done()) return;
  for (int h = h0; h < min(h0 + heads, shape.H); ++h) {
    // Rows and log-sum-exps of some runs are asked for together, a wave's share of the rows and, lane by lane, all of
    // the others; more runs come as many at a time, with a running maximum.
    float top = kNoMax, ll = 0.f, o[kPer] = {};
    const int hkv = h / shape.rep;
    Parts parts[kSides];
#pragma unroll
    for (int s = 0; s < kSides; ++s) parts[s] = token.parts(p, hkv, h - hkv * shape.rep, s);
    // (the sides' runs one after the other)
    const int runs = parts[0].runs + (kSides > 1 ? parts[kSides - 1].runs : 0);
    auto row_of = [&](int i, const float*& lse) {
      const Parts& side = kSides > 1 && i >= parts[0].runs ? parts[kSides - 1] : parts[0];
      const int64_t row = side.first + (i - (kSides > 1 && i >= parts[0].runs ? parts[0].runs : 0)) * side.step;
      lse = side.lse + row;
      return side.o + row * D;
    };
    auto some = [&](int i0, auto count) __attribute__((always_inline)) {   // runs i0 .., kShare * count of them
      fvec x[count];
      const float* at = nullptr;
#pragma unroll
      for (int k = 0; k < count; ++k) x[k] = *reinterpret_cast<const fvec*>(row_of(min(i0 + kShare * k + wave, runs - 1), at) + kPer * lane);
      row_of(min(i0 + lane, runs - 1), at);
      const float lse = i0 + lane < runs && lane < kShare * count ? *at : -INFINITY;
      float mm = lse;
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) mm = fmaxf(mm, __shfl_xor(mm, d, 64));
      mm = fmaxf(mm, top);
      const float w = fast_exp2(lse - mm), former = fast_exp2(top - mm);
      top = mm;
      ll *= former;
#pragma unroll
      for (int e = 0; e < kPer; ++e) o[e] *= former;
#pragma unroll
      for (int k = 0; k < count; ++k) {
        const float wk = lane_value(w, kShare * k + wave);   // (0 behind the last, whose row is the last one's again)
        ll += wk;
        const bool there = i0 + kShare * k + wave < runs;   // (0 times an infinity is not 0)
#pragma unroll
        for (int e = 0; e < kPer; ++e) o[e] += there ? wk * x[k][e] : 0.f;
      }
    };
    if (runs > 0 && runs <= 4 * kShare) some(0, std::integral_constant<int, 4>{});
    else if ((kShare == 1 || kShares<Table>) && runs > 0 && runs <= 8 * kShare) some(0, std::integral_constant<int, 8>{});
    else
      for (int i0 = 0; i0 < runs; i0 += 16 * kShare) some(i0, std::integral_constant<int, 16>{});
    if constexpr (kShare == 1) {
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      elem* const to = p.out + ((int64_t)t * shape.H + h) * D + kPer * lane;
      if constexpr (kPer == 2) *reinterpret_cast<uint32_t*>(to) = pack2<E>(o[0] * inv, o[1] * inv);
      else to[0] = (elem)(o[0] * inv);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) red[wave][kPer * lane + e] = o[e];
      if (lane == 0) red_l[wave] = ll;
      __syncthreads();
      if (threadIdx.x < D) {
        const int d = threadIdx.x;
        const float l4 = red_l[0] + red_l[1] + red_l[2] + red_l[3];
        p.out[((int64_t)t * shape.H + h) * D + d] = (elem)(l4 == 0.f ? 0.f : (red[0][d] + red[1][d] + red[2][d] + red[3][d]) / l4);
      }
      __syncthreads();
    }
  }
}

// The same where there are many tokens and every row is merged (kShares): `heads` heads of a token to a wave, kHeads at a time, 16 lanes to a
// head.  Finding a row's parts takes more instructions than its sums, so a lane has D / 16 elements, and its head's log-sum-exps too: 958
// tokens of 32 heads, three runs and more of each, 16 us, and 23.6 with a head to a wave.
template <class E, int D, class Table>
__global__ __launch_bounds__(256) void paged_merge_many_kernel(const PagedParams<E, Table> p, int heads) {
  static_assert(kShares<Table>);
  constexpr int kPer = D / 16, kHeads = 4, kLse = 16, kRowsAhead = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto& shape = p.shape;
  const int per_token = (shape.H + heads - 1) / heads, item = (int)blockIdx.x * 4 + wave;
  const int t = item / per_token, h0 = (item - t * per_token) * heads;
  if (t >= shape.table.T) return;
  const MergeToken<E, Table> token(p, t, lane);
  const int d0 = (lane & 15) * kPer, end = min(h0 + heads, shape.H);
  for (int h1 = h0; h1 < end; h1 += kHeads) {
    const int head = h1 + (lane >> 4), h = min(head, end - 1), hkv = h / shape.rep;   // (heads behind the last are it again)
    Parts parts[2];   // (one side's runs after the other's)
#pragma unroll
    for (int s = 0; s < 2; ++s) parts[s] = token.parts(p, hkv, h - hkv * shape.rep, s);
    const int runs = parts[0].runs + parts[1].runs;
    auto row_of = [&](int i) __attribute__((always_inline)) {
      return i >= parts[0].runs ? parts[1].first + (i - parts[0].runs) * parts[1].step : parts[0].first + i * parts[0].step;
    };
    auto side_of = [&](int i) __attribute__((always_inline)) -> const Parts& { return i >= parts[0].runs ? parts[1] : parts[0]; };
    float top = kNoMax, ll = 0.f, o[kPer] = {};
    for (int i0 = 0; __any(i0 < runs); i0 += kLse) {
      float lse[kLse], mm = top;
#pragma unroll
      for (int k = 0; k < kLse; ++k) {
        lse[k] = -INFINITY;
        if (i0 + k < runs) lse[k] = side_of(i0 + k).lse[row_of(i0 + k)];
      }
#pragma unroll
      for (int k0 = 0; k0 < kLse; k0 += kRowsAhead) {
        if (!__any(i0 + k0 < runs)) break;
        float x[kRowsAhead][kPer];
#pragma unroll
        for (int k = 0; k < kRowsAhead; ++k) {
          const int i = i0 + k0 + k;
          if (i < runs) {
            const float* const from = side_of(i).o + row_of(i) * D + d0;
#pragma unroll
            for (int e = 0; e < kPer; e += 4) {
              const f32x4 v = *reinterpret_cast<const f32x4*>(from + e);
#pragma unroll
              for (int c = 0; c < 4; ++c) x[k][e + c] = v[c];
            }
          }
        }
        if (k0 == 0) {
#pragma unroll
          for (int k = 0; k < kLse; ++k) mm = fmaxf(mm, lse[k]);
          const float former = fast_exp2(top - mm);
          top = mm;
          ll *= former;
#pragma unroll
          for (int e = 0; e < kPer; ++e) o[e] *= former;
        }
#pragma unroll
        for (int k = 0; k < kRowsAhead; ++k) {
          const float w = fast_exp2(lse[k0 + k] - mm);
          ll += w;
#pragma unroll
          for (int e = 0; e < kPer; ++e) o[e] += i0 + k0 + k < runs ? w * x[k][e] : 0.f;   // (0 times an infinity is not 0)
        }
      }
    }
    const float inv = ll == 0.f ? 0.f : 1.f / ll;
    if (head < end) {
      typename E::elem* const to = p.out + ((int64_t)t * shape.H + h) * D + d0;
#pragma unroll
      for (int e = 0; e < kPer; e += 4)
        *reinterpret_cast<u32x2*>(to + e) = u32x2{pack2<E>(o[e] * inv, o[e + 1] * inv), pack2<E>(o[e + 2] * inv, o[e + 3] * inv)};
    }
  }
}

// ---- the host's side

// Bounds of a cut's units, for any division of T tokens among B sequences of any lengths: n groups (of every sequence
// with rows, ceil(rows / group_rows)) in runs of work / left tiles are at most left + n units (run_tiles()).
static Cut bounded_cut(Cut c, int64_t T, int B, int rep) {
  // (of a cut with rows_over, at most T * rep / (rows_over + 1) sequences)
  const int64_t with_rows = c.rows_over ? T * rep / (c.rows_over + 1) : T, sequences = with_rows < B ? with_rows : B;
  // (no sequence has more groups than rows_up_to rows make)
  const int64_t by_rows = sequences + T * rep / c.group_rows, by_sequences = sequences * ((c.rows_up_to - 1) / c.group_rows + 1);
  const int64_t groups = by_rows < by_sequences ? by_rows : by_sequences;
  const int64_t several = groups < (int64_t)kWholeAt * c.target ? groups : (int64_t)kWholeAt * c.target;
  const int64_t parts = c.target / 2 + 1 + several > c.target ? c.target / 2 + 1 + several : c.target;
  const int64_t most = groups > parts ? groups : parts;
  c.parts = (int)parts;
  c.most = (int)(most < 0x7fffffff ? most : 0x7fffffff);
  return c;
}

// One round of workgroups, two to a compute unit (one where a wave's blocks are large).  Sequences of many rows per key/value head
// go to the many-row kernel, if it is launched: if there may be any.
struct Cuts {
  Cut few, many;
};
// T: rows of the batch, counted as often as they are attended; few_per_cu: workgroups of few rows
static Cuts paged_cuts(int64_t T, int sequences, int rep, int Hkv, int D, bool cache8, bool many, int group_rows, int few_rows, int few_per_cu) {
  const int cus = compute_units() > 0 ? compute_units() : 256;
  auto target = [&](int per_cu) { return per_cu * cus / Hkv > 0 ? per_cu * cus / Hkv : 1; };
  Cuts c;
  // (runs of at least two tiles: one token against 4096 keys, with the merge 13.5 us with runs of one, 12.3 of two, 13.4 of three)
  c.few = bounded_cut({group_rows, kFewTile, 2, 0, many ? few_rows : 0x7fffffff, target(few_per_cu), 0, 0, false}, T, sequences, rep);
  c.many = {};
  if (many) {
    const int waves = D == 128 && cache8 ? kManyWaves<128, true> : kManyWaves<64, false>;
    // (695 tokens and 204 against 883 and 151, 5 heads on one: 30.0 us with runs of any length, 24.4 with at least four tiles, 24.6 with
    // six; 609 tokens of 8 heads: 27.5, 21, 21)
    c.many = bounded_cut({32 * waves, kManyKeys, 4, few_rows, 0x7fffffff, target(8 / waves), 0, 0, false}, T, sequences, rep);
  }
  return c;
}

static bool paged_sizes_ok(int64_t T, int B, int H, int Hkv) {
  return T > 0 && B > 0 && H > 0 && Hkv > 0 && H % Hkv == 0;
}
static int64_t part_rows(const Cut& c, int Hkv) { return (int64_t)c.parts * Hkv * c.group_rows; }
static int64_t runs_bytes(int B) { return ((int64_t)B * sizeof(Runs) + 15) / 16 * 16; }

// The arguments that the entry points have in common: `table` filled, or an error code
static int check_paged(PageTable& table, const void* q, const void* out, const void* k_pages, const void* v_pages, const float* k_scales,
                       const float* v_scales, const int32_t* page_table, const int32_t* lengths, const int32_t* cu_new,
                       const void* workspace, int64_t T, int B, int H, int Hkv, int D, int page_size, int64_t num_pages,
                       int64_t max_pages, const int64_t* strides, int cache8, int dtype) {
  if (!q || !out || !k_pages || !v_pages || !page_table || !lengths || !cu_new || !workspace || !strides) return MOBA_ERR_ARG;
  if (!paged_sizes_ok(T, B, H, Hkv) || num_pages <= 0 || max_pages <= 0 || (cache8 && (!k_scales || !v_scales))) return MOBA_ERR_ARG;
  const int page_log2 = page_log2_of(page_size);
  if ((D != 64 && D != 128) || page_log2 < 0 || (dtype != MOBA_DTYPE_BF16 && dtype != MOBA_DTYPE_F16)) return MOBA_ERR_UNSUPPORTED;
  for (const void* x : {q, k_pages, v_pages, workspace})
    if ((uintptr_t)x & 15) return MOBA_ERR_ARG;
  if (((uintptr_t)out & 7) || (strides[0] & 7) || (strides[1] & 7)) return MOBA_ERR_ARG;  // 16-byte loads, 8-byte stores
  if (T >= 1LL << 24 || T * H >= 1LL << 31 || num_pages >= 1LL << 31 || max_pages >= 1LL << 31) return MOBA_ERR_LIMIT;
  // (keys are numbered in 32 bits, with room for the steps behind the last)
  const int64_t reachable = 0x7fff0000LL >> page_log2;
  table = {page_table, lengths, cu_new, strides[2], B, (int)T, (int)num_pages, (int)(max_pages < reachable ? max_pages : reachable),
           page_log2};
  return MOBA_OK;
}

// Of a call whose batch counts as `sequences`: false where a launch would have more threads than 32 bits number (kChooses: several launches)
template <class E, class Table>
static bool set_params(PagedParams<E, Table>& p, const Cuts& cuts, const void* q, void* out, const void* k_pages, const void* v_pages,
                       const float* k_scales, const float* v_scales, char* workspace, int sequences, int D, const int64_t* strides,
                       bool cache8, float scale) {
  typedef typename E::elem elem;
  const int Hkv = p.shape.Hkv;
  const int64_t many_threads = 64 * (D == 128 && cache8 ? kManyWaves<128, true> : kManyWaves<64, false>);
  p.few = cuts.few;
  p.many = cuts.many;
  if ((!kChooses<Table> && (int64_t)p.few.most * Hkv * 64 * kFewWaves >= 1LL << 32) || (int64_t)p.many.most * Hkv * many_threads >= 1LL << 32)
    return false;
  p.q = (const elem*)q; p.out = (elem*)out;
  p.pages[0] = (const char*)k_pages; p.pages[1] = (const char*)v_pages;
  p.scales[0] = k_scales; p.scales[1] = v_scales;
  p.runs = (Runs*)workspace;
  p.few_o = (float*)(workspace + runs_bytes(sequences));
  p.few_lse = p.few_o + part_rows(p.few, Hkv) * D;
  p.many_o = p.few_lse + part_rows(p.few, Hkv);
  p.many_lse = p.many_o + part_rows(p.many, Hkv) * D;
  p.q_tok_stride = strides[0]; p.q_head_stride = strides[1];
  p.scale_log2 = scale * 1.4426950408889634f;
  return true;
}
static size_t paged_workspace_bytes(const Cuts& c, int sequences, int Hkv, int D) {
  return (size_t)runs_bytes(sequences) + (size_t)(part_rows(c.few, Hkv) + part_rows(c.many, Hkv)) * (D + 1) * sizeof(float);
}

template <class E, int D, class Table>
static void launch_merge(const PagedParams<E, Table>& p, hipStream_t st) {
  const int64_t rows = (int64_t)p.shape.table.T * p.shape.H;
  // (a wave to a row from some thousand rows on: 774 tokens of 16 heads, five runs each, 29.7 us with four, 9.8 so; 136 of 8, up to 60
  // runs: 5.3 and 4.0; 69 of 8 and less are equal, 37 of 8, up to 256 runs: 9 with four, 16 so)
  if (rows <= 1024) {
    hipLaunchKernelGGL((paged_merge_kernel<E, D, 4, Table>), dim3((unsigned)rows), dim3(256), 0, st, p, 1);
    return;
  }
  // (kShares, four heads at a time: 40 tokens of 32 heads 1.9 us slower than a head to a wave, 128 2.3, 958 seven faster)
  const int64_t rounds = (rows + 16383) / 16384, want = kShares<Table> && rounds > 1 ? 4 * rounds : rounds;
  const int heads = (int)(want < p.shape.H ? want : p.shape.H), per_token = (p.shape.H + heads - 1) / heads;
  const dim3 grid((unsigned)(((int64_t)p.shape.table.T * per_token + 3) / 4));
  if constexpr (kShares<Table>) {
    if (rounds > 1) {
      hipLaunchKernelGGL((paged_merge_many_kernel<E, D, Table>), grid, dim3(256), 0, st, p, heads);
      return;
    }
  }
  hipLaunchKernelGGL((paged_merge_kernel<E, D, 1, Table>), grid, dim3(256), 0, st, p, heads);
}

template <class E, int D, bool k8, class Table>
static int launch_paged(const PagedParams<E, Table>& p, hipStream_t st) {
  LaunchCheck launch_check;
  static bool allowed[2][kMaxDevices];
  const auto few = paged_few_kernel<E, D, k8, Table, few_sets<Table>(D)>;
  if (!allow_dynamic_lds((const void*)few, few_lds_bytes<D, k8, Table>(), allowed[0])) return MOBA_ERR_LAUNCH;
  auto launch_few = [&](const PagedParams<E, Table>& now, int units) {
    hipLaunchKernelGGL(few, dim3((unsigned)units * now.shape.Hkv), dim3(64 * kFewWaves), (few_lds_bytes<D, k8, Table>()), st, now);
  };
  if constexpr (kChooses<Table>) {   // (a launch's lists lie where those of the one before it have been)
    PagedParams<E, Table> now = p;
    const int step = now.shape.table.units;
    for (int& unit0 = now.shape.table.unit0; unit0 < p.few.most; unit0 += step) launch_few(now, std::min(step, p.few.most - unit0));
  } else {
    launch_few(p, p.few.most);
    if (p.many.most > 0) {
      const auto many = paged_many_kernel<E, D, k8, Table>;
      if (!allow_dynamic_lds((const void*)many, many_lds_bytes<D>(), allowed[1])) return MOBA_ERR_LAUNCH;
      hipLaunchKernelGGL(many, dim3((unsigned)p.many.most * p.shape.Hkv), dim3(64 * (kManyWaves<D, k8>)), many_lds_bytes<D>(), st, p);
    }
  }
  launch_merge<E, D>(p, st);
  return launch_check.result();
}

}  // namespace moba
