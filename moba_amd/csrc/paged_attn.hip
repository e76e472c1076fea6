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
// A page's key scale multiplies the scores, its value scale the probabilities, both in 32 bits.
//
// Precision: the scores' products are exact, their sums 32 bits.  A probability (times the value scale) goes to the second product as
// the sum of two elements, its rounded value and the rounded rest (16 bits of it in bf16, 22 in fp16).
//
// Rows that see no key are zeros.  Values that are not finite reach the rows that see them and no others: a key that a row
// does not see has the probability 0, but 0 * Inf is NaN, so a wave whose sums are not finite goes through its keys again
// one by one, every row with the keys that it sees.  (Rows of a page behind the sequence's end are cleared on the way: they
// hold whatever was there.)
//
//   paged_few_kernel    one run of keys: out itself; several: part_o, part_lse (normalised, log2 domain) of every run
//   paged_merge_kernel  the runs of a row together; zeros where there is nothing to see
#include "attn_common.h"
#include "paged_cut.h"
#include <type_traits>

namespace moba {

constexpr int kFewWaves = 4;
constexpr int kFewKeys = 32;                       // of a wave's step
constexpr int kFewRows = 32;
constexpr int kFewTile = kFewWaves * kFewKeys;     // keys of a workgroup's step
constexpr int kSlot = 16;                          // keys of which a block's page is looked up together
constexpr int kBatch = 64 / (kFewKeys / kSlot);    // steps whose pages one wave looks up at a time
constexpr int kScaleBytes = 2 * 2 * 64 * 4;        // of a wave: two batches, K's and V's scales of 64 slots

template <class E>
struct PagedParams {
  typedef typename E::elem elem;
  Shape shape;
  Cut few;
  const elem* q;
  elem* out;              // [T, H, D]
  const char* pages[2];
  const float* scales[2];
  float* part_o;          // [parts * Hkv, group_rows, D]
  float* part_lse;
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

// eight e4m3 numbers as elements of a 16-bit type (exact)
__device__ __forceinline__ bf16x8 widened(uint32_t a, uint32_t b, Bf16) {
  const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, false), q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, true);
  const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, false), s = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, true);
  return bf16x8{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}
__device__ __forceinline__ f16x8 widened(uint32_t a, uint32_t b, F16) {
  const f16x2 p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, false), q = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, true);
  const f16x2 r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, false), s = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, true);
  return f16x8{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}

// fp16 probabilities are kept 2^7 times larger (the running maximum may lag by 2^8: they stay below 2^15), so that
// those far below the maximum stay above the type's smallest number; the factor cancels
template <class V> struct ProbShift { static constexpr float value = 0.f; };
template <> struct ProbShift<F16> { static constexpr float value = 7.f; };
constexpr float kMaxLag = 8.f;
constexpr float kNoMax = -3e38f;  // before the first visible key (finite: exp2(m - m_new) stays defined)

template <int D, bool k8>
constexpr int few_stage_bytes() { return 2 * kFewKeys * D * (k8 ? 1 : 2); }  // K and V of a step
template <int D, bool k8>
constexpr int few_lds_bytes() {
  const int loop = kFewWaves * (2 * few_stage_bytes<D, k8>() + kScaleBytes);
  const int end = kFewWaves * (32 * (D + 4) * 4 + 2 * 32 * 4);
  return loop > end ? loop : end;
}

template <class E, int D, bool k8>
__global__ __launch_bounds__(64 * kFewWaves, 2) void paged_few_kernel(const PagedParams<E> p) {
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
  const Shape& shape = p.shape;
  const PageTable& table = shape.table;
  const int u = (int)blockIdx.x / shape.Hkv, hkv = (int)blockIdx.x - u * shape.Hkv;

  const Share first = share_at(shape, p.few, lane);
  const int run = run_tiles(shape, p.few, lane, first);
  if (run == 0) return;   // (no work at all)
  const Unit unit = unit_at(shape, p.few, u, run, lane, first);
  if (unit.b < 0 || (unit.runs > 1 && u >= p.few.parts)) return;   // (the latter: row ranges that are none)
  const int b = __builtin_amdgcn_readfirstlane(unit.b);
  const Sequence seq = sequence_of(table, b);
  const int keys = keys_of(shape, seq);
  const int count = seq.hi - seq.lo, rows = count * shape.rep, row0 = unit.group * kFewRows;
  const int per = (unit.tiles + unit.runs - 1) / unit.runs;   // tiles of a run
  const int key_lo = __builtin_amdgcn_readfirstlane((int)min((int64_t)unit.run * per * kFewTile, (int64_t)keys));
  const int key_hi = __builtin_amdgcn_readfirstlane((int)min((int64_t)(unit.run + 1) * per * kFewTile, (int64_t)keys));
  const int row = min(row0 + n, rows - 1);   // (rows past the last repeat it and are not written)
  const int j = row / shape.rep, g = row - j * shape.rep;
  const int before = (int)seq.length - count;                          // position of the first new token
  const int limit = min(before + j, key_hi - 1);                       // the row's last visible key in this run
  const int first_masked = min(before + row0 / shape.rep, key_hi - 1); // keys up to here are visible to every row
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
  auto fetch_ids = [&](int it0) __attribute__((always_inline)) {
    const int64_t key = own_lo + (int64_t)(it0 + (lane >> 1)) * kFewTile + (lane & 1) * kSlot;
    ids = key < key_hi ? page_id(table, b, key >> table.page_log2) : -1;
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
          async_copy16_sv<true>(from, ld_off[i], to + half * kBlockBytes + (slot * kSlotCopies + i) * 1024);
      }
  };

  // Q^T operands: of step s8, lane (n, hh) holds the 8 elements of row n that its 8 elements of a key meet
  elem8 bq[kSteps];
  {
    const elem* src = p.q + (int64_t)(seq.lo + j) * p.q_tok_stride + (int64_t)(hkv * shape.rep + g) * p.q_head_stride;
#pragma unroll
    for (int s8 = 0; s8 < kSteps; ++s8)
      bq[s8] = *reinterpret_cast<const elem8*>(src + (k8 ? 32 * (s8 >> 1) + 16 * hh + 8 * (s8 & 1) : 16 * s8 + 8 * hh));
  }
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

  f32x16 oacc[kDb];
#pragma unroll
  for (int db = 0; db < kDb; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) oacc[db][e] = 0.f;
  float m_run = kNoMax, l_run = 0.f;
  uint64_t there = 0;   // the slots of the batch that have a page

  for (int it = 0; it < mine; ++it) {
    const uint32_t st = (it & 1) * kStage;
    // (the ids at hand are this batch's: the next batch's are fetched behind its last step but one)
    if (it % kBatch == 0) there = __ballot(ids >= 0);
    // this block's copies have landed (the next block's may still be in flight)
    if (it + 1 < mine) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kCopies) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    f32x16 s;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.f;
    if constexpr (k8) {
      u32x4 raw[kKReads];
#pragma unroll
      for (int i = 0; i < kKReads; ++i) raw[i] = *lds_ptr<const u32x4>(koff[i] + st);
#pragma unroll
      for (int i = 0; i < kKReads; ++i) {
        s = mfma32(widened(raw[i][0], raw[i][1], E{}), bq[2 * i], s);
        s = mfma32(widened(raw[i][2], raw[i][3], E{}), bq[2 * i + 1], s);
      }
    } else {
      elem8 ka[kKReads];
#pragma unroll
      for (int i = 0; i < kKReads; ++i) ka[i] = *lds_ptr<const elem8>(koff[i] + st);
#pragma unroll
      for (int i = 0; i < kKReads; ++i) s = mfma32(ka[i], bq[i], s);
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
                                                       lds_ptr<i32x2>(voff[0][db] + st + kSlot * j2 * kRowBytes)));
        } else {
          const velem4 x = lds_read_tr<velem4>(voff[0][db] + st + kSlot * j2 * kRowBytes);
          const velem4 y = lds_read_tr<velem4>(voff[1][db] + st + kSlot * j2 * kRowBytes);
          va[j2][db] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        }
      }
    const int key0 = own_lo + it * kFewTile;
    float vs[2] = {1.f, 1.f};
    if constexpr (k8) {
      const uint32_t at = scale_base + ((it / kBatch) & 1) * (kScaleBytes / 2) + (it % kBatch) * 8;
      const f32x2 k2 = *lds_ptr<const f32x2>(at), v2 = *lds_ptr<const f32x2>(at + 256);
      vs[0] = v2[0];
      vs[1] = v2[1];
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] *= p.scale_log2 * k2[e >> 3];
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] *= p.scale_log2;
    }
    const uint32_t has = (uint32_t)(there >> (2 * (it % kBatch))) & 3;
    const bool edge = key0 + kFewKeys - 1 > first_masked || has != 3;
    if (edge) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (key0 + 8 * (e >> 2) + 4 * hh + (e & 3) > limit || !(has & (1 << (e >> 3)))) s[e] = -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
    mx = max_xhalf(mx);
    if (__any(mx > m_run + kMaxLag)) {  // rare once the maximum has settled
      const float m_new = mx > m_run + kMaxLag ? mx : m_run;
      const float alpha = fast_exp2(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < kDb; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[db][e] *= alpha;
    }
    const float ref = m_run - ProbShift<V>::value;
    velem8 hi[2], lo[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float pe = fast_exp2(s[e] - ref);
      l_run += pe;
      if constexpr (k8) pe *= vs[e >> 3];
      const velem h = (velem)pe;
      hi[e >> 3][e & 7] = h;
      lo[e >> 3][e & 7] = (velem)(pe - (float)h);
    }
    if constexpr (k8) {
#pragma unroll
      for (int j2 = 0; j2 < 2; ++j2)
#pragma unroll
        for (int db = 0; db < kDb; ++db) va[j2][db] = widened(vraw[j2][db][0], vraw[j2][db][1], Bf16{});
    }
    if (edge) {   // keys that nobody sees: whatever lies there
#pragma unroll
      for (int j2 = 0; j2 < 2; ++j2)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (key0 + kSlot * j2 + 8 * (i >> 2) + 4 * hh + (i & 3) >= key_hi || !(has & (1 << j2))) {
#pragma unroll
            for (int db = 0; db < kDb; ++db) va[j2][db][i] = (velem)0.f;
          }
    }
#pragma unroll
    for (int j2 = 0; j2 < 2; ++j2)
#pragma unroll
      for (int db = 0; db < kDb; ++db) oacc[db] = mfma32(va[j2][db], hi[j2], oacc[db]);
#pragma unroll
    for (int j2 = 0; j2 < 2; ++j2)
#pragma unroll
      for (int db = 0; db < kDb; ++db) oacc[db] = mfma32(va[j2][db], lo[j2], oacc[db]);
    if (it + 2 < mine) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // every fragment of this stage is in registers
      issue(it + 2);
    }
  }
  if (__builtin_expect(__any(any_not_finite(oacc)), 0)) {  // (never for values of ordinary size)
    auto each_key = [&](auto use) __attribute__((always_inline)) {
      for (int it = 0; it < mine; ++it) {
        const int key0 = own_lo + it * kFewTile, key1 = min(key0 + kFewKeys, key_hi);
        for (int key = key0; key < key1; ++key) {
          const int id = __builtin_amdgcn_readfirstlane(page_id(table, b, key >> table.page_log2));
          if (id < 0) continue;
          const int64_t at = head_bytes + id * page_bytes + (key & page_mask) * kRowBytes;
          float d = 0.f, ks = 1.f, vscale = 1.f;
          if constexpr (k8) {
            ks = p.scales[0][(int64_t)id * shape.Hkv + hkv];
            vscale = p.scales[1][(int64_t)id * shape.Hkv + hkv];
          }
#pragma unroll
          for (int s8 = 0; s8 < kSteps; ++s8) {
            elem8 x;
            if constexpr (k8) {
              const u32x2 w = *reinterpret_cast<const u32x2*>(p.pages[0] + at + 32 * (s8 >> 1) + 16 * hh + 8 * (s8 & 1));
              x = widened(w[0], w[1], E{});
            } else {
              x = *reinterpret_cast<const elem8*>(p.pages[0] + at + (16 * s8 + 8 * hh) * 2);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) d += (float)bq[s8][e] * (float)x[e];
          }
          const float sc = sum_xhalf(d) * (p.scale_log2 * ks);
          if (key <= limit) use(at, sc, vscale);
        }
      }
    };
    m_run = kNoMax;
    each_key([&](int64_t, float sc, float) __attribute__((always_inline)) { m_run = fmaxf(m_run, sc); });
    const float ref = m_run - ProbShift<V>::value;
    float l = 0.f;
#pragma unroll
    for (int db = 0; db < kDb; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) oacc[db][e] = 0.f;
    each_key([&](int64_t at, float sc, float vscale) __attribute__((always_inline)) {
      float pe = fast_exp2(sc - ref);
      l += pe;
      pe *= vscale;
#pragma unroll
      for (int i = 0; i < 4 * kDb; ++i) {   // (elements 8i + 4hh .. + 3)
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
  l_run = sum_xhalf(l_run);

  // ---- the waves meet in LDS.  Element e of lane (n, hh) is O[row n][32*db + 8*(e/4) + 4*hh + e%4].
  __syncthreads();  // every wave has read its last fragments
  float* red = reinterpret_cast<float*>(smem);
  float* red_m = red + kFewWaves * 32 * kRedRow;
  float* red_l = red_m + kFewWaves * 32;
  const int rows_here = min(kFewRows, rows - row0);
  if (n < rows_here) {
#pragma unroll
    for (int db = 0; db < kDb; ++db)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4)
        *reinterpret_cast<f32x4*>(red + (wave * 32 + n) * kRedRow + 32 * db + 8 * g4 + 4 * hh) =
            f32x4{oacc[db][4 * g4], oacc[db][4 * g4 + 1], oacc[db][4 * g4 + 2], oacc[db][4 * g4 + 3]};
    if (hh == 0) {
      red_m[wave * 32 + n] = m_run;
      red_l[wave * 32 + n] = l_run;
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
    if (unit.runs == 1) {
      const int jj = (row0 + rr) / shape.rep, gg = row0 + rr - jj * shape.rep;
      const int64_t orow = (int64_t)(seq.lo + jj) * shape.H + hkv * shape.rep + gg;
      *reinterpret_cast<u32x2*>(p.out + orow * D + d) = u32x2{pack2<E>(oo[0] * inv, oo[1] * inv), pack2<E>(oo[2] * inv, oo[3] * inv)};
    } else {
      const int64_t prow = (int64_t)blockIdx.x * kFewRows + rr;
      *reinterpret_cast<f32x4*>(p.part_o + prow * D + d) = f32x4{oo[0] * inv, oo[1] * inv, oo[2] * inv, oo[3] * inv};
      if (d == 0) p.part_lse[prow] = ll == 0.f ? -INFINITY : mm - ProbShift<V>::value + fast_log2(ll);
    }
  }
}

// One workgroup per row at a time: four waves take a quarter of the runs each, a lane owns D / 64 elements; the four sums meet
// in LDS.
template <class E, int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(const PagedParams<E> p) {
  typedef typename E::elem elem;
  constexpr int kPer = D / 64;
  __shared__ float red[4][D];
  __shared__ float red_l[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Shape& shape = p.shape;
  const PageTable& table = shape.table;
  const Share first = share_at(shape, p.few, lane);
  const int run = run_tiles(shape, p.few, lane, first);
  for (int64_t row = blockIdx.x; row < (int64_t)table.T * shape.H; row += gridDim.x) {
    const int t = (int)(row / shape.H), h = (int)(row - (int64_t)t * shape.H);
    const int hkv = h / shape.rep, g = h - hkv * shape.rep;
    const int b = count_up_to(table.B, t, lane, [&](int i) { return (int64_t)table.cu_new[i + 1]; });
    int runs = 0, group = 0, groups = 0;
    int64_t unit0 = 0;
    int rr = 0;
    if (b < table.B) {
      const Sequence seq = sequence_of(table, b);
      const Share s = share_of(shape, p.few, seq);
      if (s.groups && t >= seq.lo && t < seq.hi) {
        runs = runs_of(s.tiles, run);
        groups = s.groups;
        const int r = (t - seq.lo) * shape.rep + g;
        group = r / kFewRows;
        rr = r - group * kFewRows;
        unit0 = first_unit(shape, p.few, b, run, lane, first);
      }
    }
    if (runs == 1) continue;   // (written by its one run; the same in the whole workgroup)
    if (unit0 + (int64_t)runs * groups > p.few.parts) runs = 0;   // (row ranges that are none)
    auto part = [&](int i) { return ((unit0 + (int64_t)i * groups + group) * shape.Hkv + hkv) * kFewRows + rr; };
    float mm = -INFINITY;
    for (int i = lane; i < runs; i += 64) mm = fmaxf(mm, p.part_lse[part(i)]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o, 64));
    const float top = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f, o[kPer] = {};
#pragma unroll 4
    for (int i = wave; i < runs; i += 4) {
      const int64_t at = part(i);
      const float w = fast_exp2(p.part_lse[at] - top);
      ll += w;
#pragma unroll
      for (int e = 0; e < kPer; ++e) o[e] += w * p.part_o[at * D + kPer * lane + e];
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) red[wave][kPer * lane + e] = o[e];
    if (lane == 0) red_l[wave] = ll;
    __syncthreads();
    if (threadIdx.x < D) {
      const int d = threadIdx.x;
      const float l4 = red_l[0] + red_l[1] + red_l[2] + red_l[3];
      p.out[row * D + d] = (elem)(l4 == 0.f ? 0.f : (red[0][d] + red[1][d] + red[2][d] + red[3][d]) / l4);
    }
    __syncthreads();
  }
}

}  // namespace moba

using namespace moba;

// Bounds of a cut's units, for any division of T tokens among B sequences of any lengths: n groups (of every sequence
// with rows, ceil(rows / group_rows)) in runs of work / left tiles are at most left + n units (run_tiles()).
static Cut bounded_cut(Cut c, int64_t T, int B, int rep) {
  const int64_t groups = (T < B ? T : B) + T * rep / c.group_rows;
  const int64_t several = groups < (int64_t)kWholeAt * c.target ? groups : (int64_t)kWholeAt * c.target;
  const int64_t parts = c.target / 2 + 1 + several > c.target ? c.target / 2 + 1 + several : c.target;
  const int64_t most = groups > parts ? groups : parts;
  c.parts = (int)parts;
  c.most = (int)(most < 0x7fffffff ? most : 0x7fffffff);
  return c;
}

// The cut of the few-row kernel: one round of workgroups, two to a compute unit with 8-bit pages and with narrow heads.
static Cut few_cut(int64_t T, int B, int rep, int Hkv, int D, bool cache8) {
  const int cus = compute_units() > 0 ? compute_units() : 256;
  const int slots = cus * (D == 128 && !cache8 ? 1 : 2);
  return bounded_cut({kFewRows, kFewTile, 0, 0x7fffffff, slots / Hkv > 0 ? slots / Hkv : 1, 0, 0}, T, B, rep);
}

static bool paged_sizes_ok(int64_t T, int B, int H, int Hkv) {
  return T > 0 && B > 0 && H > 0 && Hkv > 0 && H % Hkv == 0;
}
static int64_t part_rows(const Cut& c, int Hkv) { return (int64_t)c.parts * Hkv * c.group_rows; }

extern "C" size_t moba_paged_attention_workspace_bytes(int64_t T, int B, int H, int Hkv, int D, int cache8) {
  if (!paged_sizes_ok(T, B, H, Hkv) || (D != 64 && D != 128)) return 0;
  return (size_t)part_rows(few_cut(T, B, H / Hkv, Hkv, D, cache8 != 0), Hkv) * (D + 1) * sizeof(float);
}

template <class E, int D, bool k8>
static int launch_paged(const PagedParams<E>& p, hipStream_t st) {
  LaunchCheck launch_check;
  static bool allowed[kMaxDevices];
  const auto kernel = paged_few_kernel<E, D, k8>;
  if (!allow_dynamic_lds((const void*)kernel, few_lds_bytes<D, k8>(), allowed)) return MOBA_ERR_LAUNCH;
  hipLaunchKernelGGL(kernel, dim3((unsigned)p.few.most * p.shape.Hkv), dim3(64 * kFewWaves), (few_lds_bytes<D, k8>()), st, p);
  const int64_t rows = (int64_t)p.shape.table.T * p.shape.H;
  hipLaunchKernelGGL((paged_merge_kernel<E, D>), dim3((unsigned)(rows < 8192 ? rows : 8192)), dim3(256), 0, st, p);
  return launch_check.result();
}

template <class E>
static int paged_attention(const void* q, void* out, const void* k_pages, const void* v_pages, const float* k_scales,
                           const float* v_scales, const PageTable& table, float* workspace, int H, int Hkv, int D,
                           const int64_t* strides, int cache8, float scale, hipStream_t st) {
  typedef typename E::elem elem;
  PagedParams<E> p = {};
  p.shape = {table, H, Hkv, H / Hkv};
  p.few = few_cut(table.T, table.B, p.shape.rep, Hkv, D, cache8 != 0);
  if ((int64_t)p.few.most * Hkv >= 1LL << 24) return MOBA_ERR_LIMIT;   // (threads of a launch: 32 bits)
  p.q = (const elem*)q; p.out = (elem*)out;
  p.pages[0] = (const char*)k_pages; p.pages[1] = (const char*)v_pages;
  p.scales[0] = k_scales; p.scales[1] = v_scales;
  p.part_o = workspace;
  p.part_lse = workspace + part_rows(p.few, Hkv) * D;
  p.q_tok_stride = strides[0]; p.q_head_stride = strides[1];
  p.scale_log2 = scale * 1.4426950408889634f;
  if (D == 128) return cache8 ? launch_paged<E, 128, true>(p, st) : launch_paged<E, 128, false>(p, st);
  return cache8 ? launch_paged<E, 64, true>(p, st) : launch_paged<E, 64, false>(p, st);
}

// strides, in elements: {q token, q head, page table row}
extern "C" int moba_paged_attention(const void* q, void* out, const void* k_pages, const void* v_pages, const float* k_scales,
                                    const float* v_scales, const int32_t* page_table, const int32_t* lengths,
                                    const int32_t* cu_new, void* workspace, int64_t T, int B, int H, int Hkv, int D, int page_size,
                                    int64_t num_pages, int64_t max_pages, const int64_t* strides, int cache8, float scale,
                                    int dtype, void* stream) {
  if (!q || !out || !k_pages || !v_pages || !page_table || !lengths || !cu_new || !workspace || !strides) return MOBA_ERR_ARG;
  if (!paged_sizes_ok(T, B, H, Hkv) || num_pages <= 0 || max_pages <= 0 || (cache8 && (!k_scales || !v_scales))) return MOBA_ERR_ARG;
  const int page_log2 = page_log2_of(page_size);
  if ((D != 64 && D != 128) || page_log2 < 0 || (dtype != MOBA_DTYPE_BF16 && dtype != MOBA_DTYPE_F16)) return MOBA_ERR_UNSUPPORTED;
  for (const void* x : {q, k_pages, v_pages, (const void*)workspace})
    if ((uintptr_t)x & 15) return MOBA_ERR_ARG;
  if (((uintptr_t)out & 7) || (strides[0] & 7) || (strides[1] & 7)) return MOBA_ERR_ARG;  // 16-byte loads, 8-byte stores
  if (T >= 1LL << 30 || T * H >= 1LL << 31 || num_pages >= 1LL << 31 || max_pages >= 1LL << 31) return MOBA_ERR_LIMIT;
  // (keys are numbered in 32 bits, with room for the steps behind the last)
  const int64_t reachable = 0x7fff0000LL >> page_log2;
  const PageTable table = {page_table, lengths, cu_new, strides[2], B, (int)T, (int)num_pages,
                           (int)(max_pages < reachable ? max_pages : reachable), page_log2};
  hipStream_t st = (hipStream_t)stream;
  return dtype == MOBA_DTYPE_F16
             ? paged_attention<F16>(q, out, k_pages, v_pages, k_scales, v_scales, table, (float*)workspace, H, Hkv, D, strides,
                                    cache8, scale, st)
             : paged_attention<Bf16>(q, out, k_pages, v_pages, k_scales, v_scales, table, (float*)workspace, H, Hkv, D, strides,
                                     cache8, scale, st);
}
