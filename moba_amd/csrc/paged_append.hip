// New keys and values into the paged cache, keys (and queries) rotated by their positions on the way.
//
// A page that receives tokens is one workgroup's work, for all heads: its scales depend on all of its elements.  8-bit pages:
//   a   = largest finite magnitude among the page's new elements of the head (keys after the rotation, in 32 bits)
//   s   = 2^k with the smallest k >= -100 for which a <= 448 * 2^k; not less than the scale of the tokens that the page holds
//   new element = x / s to e4m3 (nearest even; beyond +-448 s, which only an infinity is: +-448; NaN stays NaN)
// and where s grew, the elements that the page holds are rounded again.  A power of two makes that exact but for elements
// that fall below e4m3's normal numbers (2^-15 of the page's range), and the division exact always.
//
// Bound by memory for prompts (each element is read once from memory; the second reading, after the page's maximum is known,
// comes from L2), by latency for single tokens: the angles of the page's tokens are made once for all heads, by all
// waves, and wait in LDS.
#include "paged.h"
#include "rotary.h"

namespace moba {

constexpr int kAppendWaves = 8;
constexpr int kAngleTokens = 64;   // tokens whose angles lie in LDS at a time
constexpr int kQueryTokens = 16;   // tokens of a workgroup that rotates queries
constexpr int kMostHeads = 256;    // key/value heads

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
  int H, Hkv, rotary, interleaved, items;
};

// the smallest power of two s with a <= 448 s
__device__ __forceinline__ float page_scale(float a) {
  const uint32_t bits = float_bits(a);
  const int k = (int)(bits >> 23) - 126 - 9 + ((bits & 0x7fffff) > 0x600000);   // (a denormal ends at the least exponent)
  return __builtin_bit_cast(float, (uint32_t)(max(k, kLeastScaleExponent) + 127) << 23);
}

__device__ __forceinline__ float to_e4m3_range(float x) {
  return x != x ? x : __builtin_amdgcn_fmed3f(x, -kE4m3Max, kE4m3Max);
}
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(to_e4m3_range(a), to_e4m3_range(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(to_e4m3_range(c), to_e4m3_range(d), w, true);
}
__device__ __forceinline__ void store_row8(char* row, const RowPlace& p, const float (&x)[8], float over) {
  *reinterpret_cast<uint32_t*>(row + p.a) = pack_e4m3(x[0] * over, x[1] * over, x[2] * over, x[3] * over);
  *reinterpret_cast<uint32_t*>(row + p.b) = pack_e4m3(x[4] * over, x[5] * over, x[6] * over, x[7] * over);
}
// the elements of a word as they would be with a scale 1 / by times as large
__device__ __forceinline__ uint32_t rescaled(uint32_t w, float by) {
  return pack_e4m3(__builtin_amdgcn_cvt_f32_fp8(w, 0) * by, __builtin_amdgcn_cvt_f32_fp8(w, 1) * by,
                   __builtin_amdgcn_cvt_f32_fp8(w, 2) * by, __builtin_amdgcn_cvt_f32_fp8(w, 3) * by);
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

template <class E, int D, bool k8>
__global__ __launch_bounds__(64 * kAppendWaves) void paged_append_kernel(const AppendParams<E> p) {
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

  if ((int)blockIdx.x >= p.items) {  // ---- queries: kQueryTokens tokens, all heads
    const int t0 = ((int)blockIdx.x - p.items) * kQueryTokens, count = min(kQueryTokens, table.T - t0);
    for (int i = wave; i < count; i += kAppendWaves) {
      const int b = count_up_to(table.B, t0 + i, lane, [&](int j) { return (int64_t)table.cu_new[j + 1]; });
      if (lane == 0) place[i] = b < table.B ? (int64_t)table.lengths[b] - table.cu_new[b + 1] + t0 + i : INT64_MIN;
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
  // (cu_new[b] >> page_log2) + 2b on, at least as many as its tokens can touch
  const int item = blockIdx.x;
  auto first_item = [&](int b) { return (int64_t)(min(max(table.cu_new[b], 0), table.T) >> table.page_log2) + 2 * b; };
  const int b = count_up_to(table.B, item, lane, first_item) - 1;
  if (b < 0) return;
  const Sequence seq = sequence_of(table, b);
  const int64_t begin = seq.length - (seq.hi - seq.lo);   // position of row seq.lo
  const int64_t page = (max(begin, (int64_t)0) >> table.page_log2) + (item - first_item(b));
  const int64_t first = page << table.page_log2;
  const int from = (int)(max(begin, first) - first);      // the page's new tokens: from .. to - 1
  const int to = (int)min(seq.length - first, (int64_t)1 << table.page_log2);
  if (seq.hi == seq.lo || to <= from) return;
  const int id = page_id(table, b, page);
  if (id < 0) return;
  const int64_t row_of_first = seq.lo - begin + first;    // row of the page's token 0, were it new
  const int count = to - from;
  constexpr int kBytes = k8 ? 1 : 2;
  const int64_t page_bytes = ((int64_t)p.Hkv << table.page_log2) * D * kBytes;

  for (int i = tid; i < 2 * p.Hkv; i += 64 * kAppendWaves) most[i >= p.Hkv][i >= p.Hkv ? i - p.Hkv : i] = 0;
  const bool in_pieces = count > kAngleTokens;
  for (int pass = k8 ? 0 : 1; pass < 2; ++pass) {
    for (int c0 = 0; c0 < count; c0 += kAngleTokens) {
      const int piece = min(kAngleTokens, count - c0);
      if (pass == (k8 ? 0 : 1) || in_pieces) {
        __syncthreads();   // (the angles before have been read)
        make_angles(piece, [&](int i) { return first + from + c0 + i; });
        __syncthreads();
      }
      for (int r = row0; r < piece * p.Hkv; r += kStep) {
        const int i = r / p.Hkv, h = r - i * p.Hkv;
        const int token = from + c0 + i;
        const int64_t row = row_of_first + token;
        float x[2][8];
#pragma unroll
        for (int half = 0; half < 2; ++half)
          load_row<E>(p.x[half] + row * p.tok_stride[half] + h * p.head_stride[half], at, x[half]);
        turn_row(x[0], turn_from(angles, i, u, at.turned), p.interleaved);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (pass == 0) {
            float m = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float a = fabsf(x[half][e]);
              m = fmaxf(m, a < INFINITY ? a : 0.f);
            }
#pragma unroll
            for (int o = 1; o < G; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
            if (u == 0) atomicMax(&most[half][h], float_bits(m));
          } else {
            char* to_row = p.pages[half] + id * page_bytes + (((int64_t)h << table.page_log2) + token) * (D * kBytes);
            if constexpr (k8) store_row8(to_row, at, x[half], over[half][h]);
            else store_row<E>((typename E::elem*)to_row, at, x[half]);
          }
        }
      }
    }
    if (pass == 1) break;
    __syncthreads();   // the maxima are complete
    for (int i = tid; i < 2 * p.Hkv; i += 64 * kAppendWaves) {
      const int half = i >= p.Hkv, h = half ? i - p.Hkv : i;
      float* scale = p.scales[half] + (int64_t)id * p.Hkv + h;
      const float former = from > 0 ? *scale : 0.f;
      const float s = fmaxf(page_scale(__builtin_bit_cast(float, most[half][h])), former);
      over[half][h] = 1.f / s;
      again[half][h] = former > 0.f && s > former ? former / s : 0.f;
      *scale = s;
    }
    __syncthreads();
    // tokens that the page holds, where a scale grew
    for (int r = row0; r < from * p.Hkv; r += kStep) {
      const int i = r / p.Hkv, h = r - i * p.Hkv;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float by = again[half][h];
        if (by == 0.f) continue;
        u32x2* w = reinterpret_cast<u32x2*>(p.pages[half] + id * page_bytes + (((int64_t)h << table.page_log2) + i) * D + 8 * u);
        u32x2 v = *w;
        v[0] = rescaled(v[0], by);
        v[1] = rescaled(v[1], by);
        *w = v;
      }
    }
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
  const int64_t workgroups = items + (q ? (table.T + kQueryTokens - 1) / kQueryTokens : 0);
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
