// New keys and values into the paged cache, keys (and queries) rotated by their positions on the way.
//
// A page that receives tokens is one workgroup's work, for all heads: its scales depend on all of its elements.  8-bit pages:
//   a   = largest finite magnitude among the page's new elements of the head (keys after the rotation, in 32 bits)
//   s   = 2^k with the smallest k >= -100 for which a <= 448 * 2^k; not less than the scale of the tokens that the page holds
//   new element = x / s to e4m3 (nearest even; beyond +-448 s, which only an infinity is: +-448; NaN stays NaN)
// and where s grew, the elements that the page holds are rounded again.  A power of two makes that exact but for elements
// that fall below e4m3's normal numbers (2^-15 of the page's range), and the division exact always.
//
// Bound by memory for prompts, by latency for single tokens.  The angles of the page's tokens are made once for all heads, by
// all waves, and wait in LDS; the rows go by groups of heads, two rows to a lane, which stay in registers, turned, until the
// group's maxima are known, while the next group's are on their way (read again instead, from L2 or memory, a prompt of
// 131072 tokens took 640 us).  That prompt, 32 and 8 heads, with its queries: 2.95 GB in 595 us, 5.0 TB/s; sixteen sequences of
// one new token: 6.9 us, a chain of lookup, row, maxima, the page's earlier tokens.
#include "paged.h"
#include "rotary.h"

namespace moba {

constexpr int kAppendWaves = 8;
constexpr int kAngleTokens = 64;   // tokens whose angles lie in LDS at a time
constexpr int kQueryTokens = 16;   // tokens of a workgroup that rotates queries, at most
constexpr int kMostHeads = 256;    // key/value heads
constexpr int kKeep = 2;           // rows of a lane that stay in registers between the two passes

template <class E>
struct AppendParams {
  typedef typename E::elem elem;
  PageTable table;
  const elem* x[2];      // k and v
  const elem* q;
  elem* yq;              // [T, H, D]
  char* pages[2];
  float* scales[2];      // 8-bit pages
  const float* inv_freq;
  int64_t tok_stride[2], head_stride[2], q_tok_stride, q_head_stride;
  int H, Hkv, rotary, interleaved;
  int items, query_tokens;  // pages; tokens of a workgroup that rotates queries
};

// the smallest power of two s with a <= 448 s
__device__ __forceinline__ float page_scale(float a) {
  const uint32_t bits = float_bits(a);
  const int k = (int)(bits >> 23) - 126 - 9 + ((bits & 0x7fffff) > 0x600000);   // (a denormal ends at the least exponent)
  return __builtin_bit_cast(float, (uint32_t)(max(k, kLeastScaleExponent) + 127) << 23);
}

// four numbers of that range, or NaN, to e4m3 (the instruction makes NaN of what lies beyond it)
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
__device__ __forceinline__ void store_row8(char* row, const RowPlace& p, const float (&x)[8], float over) {
  *reinterpret_cast<uint32_t*>(row + p.a) = pack_e4m3(x[0] * over, x[1] * over, x[2] * over, x[3] * over);
  *reinterpret_cast<uint32_t*>(row + p.b) = pack_e4m3(x[4] * over, x[5] * over, x[6] * over, x[7] * over);
}
// the largest finite magnitude of a lane's elements, and whether there is an infinity among them (then clamped to the type's largest
// number, which no finite element's quotient by its scale exceeds).  (The maximum passes over NaN.)
__device__ __forceinline__ float largest(const float (&x)[8], bool& infinite) {
  float m = fabsf(x[0]);
#pragma unroll
  for (int e = 1; e < 8; ++e) m = fmaxf(m, fabsf(x[e]));
  infinite = m == INFINITY;
  if (__builtin_expect(infinite, 0)) {
    m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.f);
  }
  return m == m ? m : 0.f;
}
// the elements of a word as they would be with a scale 1 / by times as large
__device__ __forceinline__ uint32_t rescaled(uint32_t w, float by) {
  return pack_e4m3(__builtin_amdgcn_cvt_f32_fp8(w, 0) * by, __builtin_amdgcn_cvt_f32_fp8(w, 1) * by,
                   __builtin_amdgcn_cvt_f32_fp8(w, 2) * by, __builtin_amdgcn_cvt_f32_fp8(w, 3) * by);
}

// the largest of a value over the G lanes of a row, in every one of them
template <int G>
__device__ __forceinline__ float row_max(float x) {
#define MOBA_DPP_MAX(ctrl) x = fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, (int)float_bits(x), ctrl, 0xf, 0xf, false)))
  MOBA_DPP_MAX(0xB1);
  MOBA_DPP_MAX(0x4E);
  MOBA_DPP_MAX(0x141);
  if constexpr (G == 16) MOBA_DPP_MAX(0x140);
#undef MOBA_DPP_MAX
  return x;
}

struct Angles {
  float2 cs[kAngleTokens][64];
};
__device__ __forceinline__ Turn turn_from(const Angles& a, int token, int u, bool turned) {
  Turn t;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = a.cs[token][(4 * u + i) & 63];
    t.c[i] = v.x;
    t.s[i] = v.y;
  }
  t.turned = turned;
  return t;
}

// a lane's two groups of a row, as they are in memory
template <class E>
__device__ __forceinline__ u32x4 load_raw(const typename E::elem* row, const RowPlace& p) {
  const u32x2 a = *reinterpret_cast<const u32x2*>(row + p.a), b = *reinterpret_cast<const u32x2*>(row + p.b);
  return u32x4{a[0], a[1], b[0], b[1]};
}
template <class E>
__device__ __forceinline__ void unpack(const u32x4& w, float (&x)[8]) {
  const typename E::elem8 v = __builtin_bit_cast(typename E::elem8, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
}

template <class E, int D, bool k8>
__global__ __launch_bounds__(64 * kAppendWaves, 4) void paged_append_kernel(const AppendParams<E> p) {
  constexpr int G = D / 8, kRows = 64 / G;       // lanes of a row, rows of a wave
  constexpr int kStep = kAppendWaves * kRows;    // rows of the workgroup
  __shared__ Angles angles;
  __shared__ uint32_t most[2][kMostHeads];       // bits of the largest magnitudes
  __shared__ float over[2][kMostHeads], again[2][kMostHeads];
  __shared__ int64_t place[kQueryTokens];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int u = lane % G, row0 = wave * kRows + lane / G;
  const RowPlace at = row_place(u, D, p.rotary, p.interleaved);
  const PageTable& table = p.table;

  auto make_angles = [&](int count, auto position) __attribute__((always_inline)) {
    for (int i = wave; i < count; i += kAppendWaves) {
      float c = 1.f, s = 0.f;
      if (2 * lane < p.rotary) turn_of((double)position(i), p.inv_freq[lane], c, s);
      angles.cs[i][lane] = float2{c, s};
    }
  };

  if ((int)blockIdx.x >= p.items) {  // ---- queries: all heads of some tokens
    const int t0 = ((int)blockIdx.x - p.items) * p.query_tokens, count = min(p.query_tokens, table.T - t0);
    for (int i = wave; i < count; i += kAppendWaves) {
      Sequence seq;
      const int b = last_up_to(table, t0 + i, lane, seq, [](int, int lo) { return (int64_t)lo; });
      if (lane == 0) place[i] = b >= 0 && t0 + i < seq.hi ? seq.length - seq.hi + t0 + i : INT64_MIN;
    }
    __syncthreads();
    make_angles(count, [&](int i) { return place[i]; });
    __syncthreads();
    for (int r = row0; r < count * p.H; r += kStep) {
      const int i = r / p.H, h = r - i * p.H;
      float x[8] = {};
      if (place[i] != INT64_MIN) {   // (rows of no sequence: zeros)
        load_row<E>(p.q + (int64_t)(t0 + i) * p.q_tok_stride + h * p.q_head_stride, at, x);
        turn_row(x, turn_from(angles, i, u, at.turned), p.interleaved);
      }
      store_row<E>(p.yq + ((int64_t)(t0 + i) * p.H + h) * D, at, x);
    }
    return;
  }

  // ---- a page: which sequence's, and which of the pages that its new tokens touch.  Sequence b's take the items from
  // (first row >> page_log2) + 2b on, at least as many as its tokens can touch
  const int item = blockIdx.x, heads = p.Hkv;
  auto first_item = [&](int b, int lo) { return (int64_t)(lo >> table.page_log2) + 2 * b; };
  Sequence seq = {0, 0, 0};
  const int b = last_up_to(table, item, lane, seq, first_item);
  if (b < 0 || seq.hi == seq.lo) return;
  const int64_t begin = seq.length - (seq.hi - seq.lo);   // position of row seq.lo
  const int64_t page = (max(begin, (int64_t)0) >> table.page_log2) + (item - first_item(b, seq.lo));
  const int64_t first = page << table.page_log2;
  const int from = (int)(max(begin, first) - first);      // the page's new tokens: from .. to - 1
  const int to = (int)min(seq.length - first, (int64_t)1 << table.page_log2);
  if (to <= from) return;
  const int count = to - from, piece0 = min(kAngleTokens, count);
  const int64_t row_of_first = seq.lo - begin + first;    // row of the page's token 0, were it new
  const typename E::elem* const source[2] = {p.x[0] + (row_of_first + from) * p.tok_stride[0],
                                             p.x[1] + (row_of_first + from) * p.tok_stride[1]};
  auto raw = [&](int half, int i, int h) __attribute__((always_inline)) {   // token `from` + i, head h
    return load_raw<E>(source[half] + i * p.tok_stride[half] + h * p.head_stride[half], at);
  };
  // Pages with up to kAngleTokens new tokens go by groups of heads whose rows stay in registers, the next group's on their way
  // (the first while the page is looked up and the angles are made).
  const bool in_pieces = !k8 || count > kAngleTokens;
  const int group = in_pieces ? heads : min(heads, max(kKeep * kStep / count, 1));
  u32x4 coming[kKeep][2];
  auto load_group = [&](int h0) __attribute__((always_inline)) {
    const int n = min(group, heads - h0);
#pragma unroll
    for (int s = 0; s < kKeep; ++s) {
      const int r = row0 + s * kStep, i = r / n;
      if (r < count * n) {
        coming[s][0] = raw(0, i, h0 + r - i * n);
        coming[s][1] = raw(1, i, h0 + r - i * n);
      }
    }
  };
  if (!in_pieces) load_group(0);
  const int id = page_id(table, b, page);
  if (id < 0) return;
  constexpr int kBytes = k8 ? 1 : 2;
  const int64_t page_bytes = ((int64_t)p.Hkv << table.page_log2) * D * kBytes;
  char* const target[2] = {p.pages[0] + id * page_bytes, p.pages[1] + id * page_bytes};
  auto row_at = [&](int half, int token, int h) { return target[half] + ((h << table.page_log2) + token) * (D * kBytes); };

  float former = 0.f;   // thread i: the scale of half i / heads, head i % heads, if the page holds tokens
  float* scale = nullptr;
  if constexpr (k8) {
    if (tid < 2 * heads) {
      const int half = tid >= heads, h = half ? tid - heads : tid;
      scale = p.scales[half] + (int64_t)id * heads + h;
      if (from > 0) former = *scale;
      most[half][h] = 0;
    }
  }
  auto turned = [&](const u32x4 (&w)[2], int i, float (&x)[2][8]) __attribute__((always_inline)) {
    unpack<E>(w[0], x[0]);
    unpack<E>(w[1], x[1]);
    if (at.turned) turn_row(x[0], turn_from(angles, i, u, true), p.interleaved);
  };
  auto add_most = [&](const float (&x)[2][8], int h) __attribute__((always_inline)) {   // whether there are infinities
    bool infinite[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const float m = row_max<G>(largest(x[half], infinite[half]));
      if (u == 0) atomicMax(&most[half][h], float_bits(m));
    }
    return infinite[0] || infinite[1];
  };
  auto put = [&](float (&x)[2][8], int token, int h, bool infinite) __attribute__((always_inline)) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if constexpr (k8) {
        float by = over[half][h];
        if (__builtin_expect(infinite, 0)) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x[half][e] = fabsf(x[half][e]) == INFINITY ? copysignf(kE4m3Max, x[half][e]) : x[half][e] * by;
          by = 1.f;
        }
        store_row8(row_at(half, token, h), at, x[half], by);
      } else {
        store_row<E>((typename E::elem*)row_at(half, token, h), at, x[half]);
      }
    }
  };
  // the scales of n heads from h0 on, from the maxima; the tokens that the page holds, where a scale grew
  auto set_scales = [&](int h0, int n) __attribute__((always_inline)) {
    __syncthreads();   // the maxima are complete
    const int half = tid >= heads, h = half ? tid - heads : tid;
    if (scale && h >= h0 && h < h0 + n) {
      // (a former scale that is none of page_scale()'s may have either sign)
      const float least = page_scale(__builtin_bit_cast(float, most[half][h]));
      const float s = fabsf(former) >= least ? former : least;
      over[half][h] = 1.f / s;
      again[half][h] = former / s;   // 1: as they are; 0: the least magnitude, or a former scale of 0
      *scale = s;
    }
    __syncthreads();
    for (int r = row0; r < from * n; r += kStep) {
      const int i = r / n, hr = h0 + r - i * n;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const float by = again[v][hr];
        if (by == 1.f) continue;
        u32x2* w = reinterpret_cast<u32x2*>(row_at(v, i, hr) + 8 * u);
        u32x2 bytes = *w;
        bytes[0] = rescaled(bytes[0], by);
        bytes[1] = rescaled(bytes[1], by);
        *w = bytes;
      }
    }
  };

  if (!in_pieces) {
    __syncthreads();   // (the maxima are cleared)
    if (p.rotary) make_angles(count, [&](int i) { return first + from + i; });
    __syncthreads();
    for (int h0 = 0; h0 < heads; h0 += group) {
      const int n = min(group, heads - h0);
      float x[kKeep][2][8];
      bool infinite[kKeep];
#pragma unroll
      for (int s = 0; s < kKeep; ++s) {
        const int r = row0 + s * kStep;
        if (r < count * n) turned(coming[s], r / n, x[s]);
      }
      if (h0 + group < heads) load_group(h0 + group);
#pragma unroll
      for (int s = 0; s < kKeep; ++s) {
        const int r = row0 + s * kStep;
        if (r < count * n) infinite[s] = add_most(x[s], h0 + r % n);
      }
      set_scales(h0, n);
#pragma unroll
      for (int s = 0; s < kKeep; ++s) {
        const int r = row0 + s * kStep;
        if (r < count * n) put(x[s], from + r / n, h0 + r % n, infinite[s]);
      }
    }
    return;
  }
  // 16-bit pages: once through the rows.  Larger 8-bit pages: twice, the angles again for every piece
  for (int pass = k8 ? 0 : 1; pass < 2; ++pass) {
    for (int c0 = 0; c0 < count; c0 += kAngleTokens) {
      const int piece = min(kAngleTokens, count - c0);
      __syncthreads();   // (the angles before have been read; the maxima are cleared)
      if (p.rotary) make_angles(piece, [&](int i) { return first + from + c0 + i; });
      __syncthreads();
      for (int r = row0; r < piece * heads; r += kStep) {
        const int i = r / heads, h = r - i * heads;
        const u32x4 w[2] = {raw(0, c0 + i, h), raw(1, c0 + i, h)};
        float x[2][8];
        turned(w, i, x);
        if (k8 && pass == 0) add_most(x, h);
        else put(x, from + c0 + i, h, k8);
      }
    }
    if (k8 && pass == 0) set_scales(0, heads);
  }
}

}  // namespace moba

using namespace moba;

template <class E, int D, bool k8>
static int launch_append(const AppendParams<E>& p, int64_t workgroups, hipStream_t st) {
  LaunchCheck launch_check;
  hipLaunchKernelGGL((paged_append_kernel<E, D, k8>), dim3((unsigned)workgroups), dim3(64 * kAppendWaves), 0, st, p);
  return launch_check.result();
}

template <class E>
static int append(const void* k, const void* v, const void* q, void* yq, void* k_pages, void* v_pages, float* k_scales,
                  float* v_scales, const PageTable& table, const float* inv_freq, int H, int Hkv, int D, int rotary,
                  const int64_t* strides, int cache8, int interleaved, hipStream_t st) {
  typedef typename E::elem elem;
  AppendParams<E> p = {};
  p.table = table;
  p.x[0] = (const elem*)k; p.x[1] = (const elem*)v; p.q = (const elem*)q; p.yq = (elem*)yq;
  p.pages[0] = (char*)k_pages; p.pages[1] = (char*)v_pages; p.scales[0] = k_scales; p.scales[1] = v_scales;
  p.inv_freq = inv_freq; p.rotary = rotary; p.interleaved = interleaved != 0; p.H = H; p.Hkv = Hkv;
  p.q_tok_stride = strides[0]; p.q_head_stride = strides[1];
  p.tok_stride[0] = strides[2]; p.head_stride[0] = strides[3];
  p.tok_stride[1] = strides[4]; p.head_stride[1] = strides[5];
  const int64_t items = (table.T >> table.page_log2) + 2LL * table.B;
  const int step = kAppendWaves * 512 / D;   // rows
  // queries: a step of the workgroup at least, sixteen tokens where there are many
  const int64_t least = H > 0 ? (step + H - 1) / H : 1, many = H > 0 ? (int64_t)table.T * H / (step * 2048) : 1;
  const int64_t tokens = many > least ? many : least;
  p.query_tokens = (int)(tokens < kQueryTokens ? tokens : kQueryTokens);
  const int64_t workgroups = items + (q ? (table.T + p.query_tokens - 1) / p.query_tokens : 0);
  if (workgroups >= 1LL << 23) return MOBA_ERR_LIMIT;   // (threads of a launch: 32 bits)
  p.items = (int)items;
  if (D == 128) return cache8 ? launch_append<E, 128, true>(p, workgroups, st) : launch_append<E, 128, false>(p, workgroups, st);
  return cache8 ? launch_append<E, 64, true>(p, workgroups, st) : launch_append<E, 64, false>(p, workgroups, st);
}

// strides, in elements: {q token, q head, k token, k head, v token, v head, page table row}
extern "C" int moba_paged_append(const void* k, const void* v, const void* q, void* yq, void* k_pages, void* v_pages,
                                 float* k_scales, float* v_scales, const int32_t* page_table, const int32_t* lengths,
                                 const int32_t* cu_new, const float* inv_freq, int64_t T, int B, int H, int Hkv, int D, int rotary,
                                 int page_size, int64_t num_pages, int64_t max_pages, const int64_t* strides, int cache8,
                                 int interleaved, int dtype, void* stream) {
  if (!k || !v || !k_pages || !v_pages || !page_table || !lengths || !cu_new || !strides) return MOBA_ERR_ARG;
  if ((q && (!yq || H <= 0)) || (rotary > 0 && !inv_freq) || (cache8 && (!k_scales || !v_scales))) return MOBA_ERR_ARG;
  if (T <= 0 || B <= 0 || Hkv <= 0 || rotary < 0 || rotary > D || (rotary & 7) || num_pages <= 0 || max_pages <= 0) return MOBA_ERR_ARG;
  const int page_log2 = page_log2_of(page_size);
  if ((D != 64 && D != 128) || page_log2 < 0 || (dtype != MOBA_DTYPE_BF16 && dtype != MOBA_DTYPE_F16)) return MOBA_ERR_UNSUPPORTED;
  for (const void* x : {k, v, q, (const void*)yq, (const void*)k_pages, (const void*)v_pages})
    if ((uintptr_t)x & 7) return MOBA_ERR_ARG;
  for (int i = 0; i < 6; ++i)
    if (strides[i] & 3) return MOBA_ERR_ARG;  // 8-byte loads
  if (T >= 1LL << 30 || num_pages >= 1LL << 31 || max_pages >= 1LL << 31 || Hkv > kMostHeads || H > (1 << 16)) return MOBA_ERR_LIMIT;
  const PageTable table = {page_table, lengths, cu_new, strides[6], B, (int)T, (int)num_pages, (int)max_pages, page_log2};
  hipStream_t st = (hipStream_t)stream;
  return dtype == MOBA_DTYPE_F16
             ? append<F16>(k, v, q, yq, k_pages, v_pages, k_scales, v_scales, table, inv_freq, H, Hkv, D, rotary, strides, cache8,
                           interleaved, st)
             : append<Bf16>(k, v, q, yq, k_pages, v_pages, k_scales, v_scales, table, inv_freq, H, Hkv, D, rotary, strides, cache8,
                            interleaved, st);
}
