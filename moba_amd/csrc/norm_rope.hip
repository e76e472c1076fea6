// Norm and rotation of query and key heads, forward and backward.
//
//   y = R(x * r * w),  r = 1 / sqrt(mean(x^2) + eps),  R the rotation by the token's position (rotary.h)
//   u = R^T dy,  n = x * r:  dx = r * (u*w - n * mean(u*w*n)),  dw = sum over tokens and heads of u * n
//
// Without a weight a side is rotated only.  Everything between the loads and the one rounding of the result is 32 bits.
//
// Bound by memory: 4 bytes an element forward, 6 backward (x is read again: its mean square is a few instructions and
// spares a saved copy).  A wave takes a token, makes the token's angles once for all of its heads, and goes through
// them 4 or 8 rows at a time, the next ones on their way meanwhile; with few tokens several waves share a token's heads.
// 131072 tokens, 40 heads of 128: 2.68 GB in 0.49 ms, 5.5 TB/s, what a copy reaches; 20480 tokens, 10 heads: 105 MB in 24.6 us
// forward, 157 MB in 38.2 backward and 3.9 for the weights' sums; one token: 3.6.
#include "rotary.h"
#include <type_traits>

namespace moba {

template <class E>
struct NormRopeParams {
  typedef typename E::elem elem;
  const elem* x[2];   // q and k
  const elem* dy[2];  // backward, packed
  elem* y[2];         // y, or dx; packed
  const void* w[2];   // elem or float, or null
  const void* positions;
  const float* inv_freq;
  float* partials;    // backward: [workgroups, 2, D]
  int64_t S, tok_stride[2], head_stride[2];
  int heads[2];
  int D, rotary, parts;
  float eps;
  int position64, w32, interleaved;
};

template <class E>
__device__ __forceinline__ void load_weight(const NormRopeParams<E>& p, int side, const RowPlace& at, float (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (!p.w[side] || !at.active) return;
  if (!p.w32) {
    load_row<E>((const typename E::elem*)p.w[side], at, w);
  } else {
    const float* f = (const float*)p.w[side];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = f[at.a + i];
      w[i + 4] = f[at.b + i];
    }
  }
}

template <class E>
__device__ __forceinline__ double position_of(const NormRopeParams<E>& p, int64_t t) {
  return p.position64 ? (double)((const int64_t*)p.positions)[t] : (double)((const int32_t*)p.positions)[t];
}

constexpr int kNormWaves = 4;
constexpr int kNormResident = 8;  // workgroups of the forward kernel that a compute unit holds

// A wave's way through its work: pieces (a token, or one of `parts` shares of its rows), and of each the steps of 64 / G rows,
// first the queries', then the keys'.  The rows of the next step are requested before the present one is worked on, and with
// a piece's first step the position of its token.
template <class E, int G, bool kBackward>
struct Walk {
  static constexpr int kRows = 64 / G;
  const NormRopeParams<E>& p;
  const RowPlace& at;
  const int lane, q_steps, steps;
  const int64_t pieces;
  struct Rows {
    u32x4 x, d;   // backward: d of dy
  };
  struct Place {
    int64_t piece, t;
    int step;
  };
  __device__ Walk(const NormRopeParams<E>& p_, const RowPlace& at_, int lane_)
      : p(p_), at(at_), lane(lane_), q_steps((p_.heads[0] + kRows - 1) / kRows),
        steps((p_.heads[0] + kRows - 1) / kRows + (p_.heads[1] + kRows - 1) / kRows), pieces(p_.S * p_.parts) {}
  __device__ __forceinline__ Place first(int64_t piece) const {
    const int64_t t = p.parts == 1 ? piece : piece / p.parts;
    return {piece, t, (int)(piece - t * p.parts)};
  }
  __device__ __forceinline__ int side(const Place& w) const { return w.step >= q_steps; }
  __device__ __forceinline__ int head(const Place& w) const {
    return (w.step - (w.step >= q_steps ? q_steps : 0)) * kRows + lane / G;
  }
  __device__ __forceinline__ Rows load(const Place& w) const {
    Rows r = {};
    const int s = side(w), h = head(w);
    if (w.piece < pieces && at.active && h < p.heads[s]) {
      auto raw = [&](const typename E::elem* row) {
        const u32x2 a = *reinterpret_cast<const u32x2*>(row + at.a), b = *reinterpret_cast<const u32x2*>(row + at.b);
        return u32x4{a[0], a[1], b[0], b[1]};
      };
      if (!kBackward || p.w[s]) r.x = raw(p.x[s] + w.t * p.tok_stride[s] + h * p.head_stride[s]);
      if constexpr (kBackward) r.d = raw(p.dy[s] + (w.t * p.heads[s] + h) * p.D);
    }
    return r;
  }
  __device__ __forceinline__ double position(const Place& w) const { return w.piece < pieces ? position_of(p, w.t) : 0.; }
};
template <class E>
__device__ __forceinline__ void unpack(const u32x4& w, float (&x)[8]) {
  const typename E::elem8 v = __builtin_bit_cast(typename E::elem8, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
}
// Every lane makes one pair's angle (of up to 64) and the lanes of a row fetch theirs.
__device__ __forceinline__ Turn lane_turn(double position, float inv_freq, int u, bool turned) {
  float c, s;
  turn_of(position, inv_freq, c, s);
  Turn t;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t.c[i] = __shfl(c, (4 * u + i) & 63, 64);
    t.s[i] = __shfl(s, (4 * u + i) & 63, 64);
  }
  t.turned = turned;
  return t;
}

template <class E, int G>
__global__ __launch_bounds__(64 * kNormWaves) void norm_rope_kernel(const NormRopeParams<E> p) {
  const int lane = threadIdx.x & 63, u = lane % G;
  const RowPlace at = row_place(u, p.D, p.rotary, p.interleaved);
  const Walk<E, G, false> walk(p, at, lane);
  const int64_t stride = (int64_t)gridDim.x * kNormWaves;
  auto here = walk.first((int64_t)blockIdx.x * kNormWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
  if (here.piece >= walk.pieces) return;
  auto rows = walk.load(here);
  double position = walk.position(here);
  const float inv_freq = 2 * lane < p.rotary ? p.inv_freq[lane] : 0.f;
  float w[2][8];
  load_weight(p, 0, at, w[0]);
  load_weight(p, 1, at, w[1]);
  const float over = 1.f / p.D;
  while (here.piece < walk.pieces) {
    const Turn turn = lane_turn(position, inv_freq, u, at.turned);
    const int64_t piece = here.piece;
    do {
      auto next = here;
      next.step += p.parts;
      if (next.step >= walk.steps) next = walk.first(here.piece + stride);
      const auto next_rows = walk.load(next);
      if (next.piece != piece) position = walk.position(next);
      const int side = walk.side(here), h = walk.head(here);
      float v[8];
      unpack<E>(rows.x, v);
      if (p.w[side]) {
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sq += v[i] * v[i];
        const float r = 1.f / sqrtf(row_sum<G>(sq) * over + p.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * r * (side ? w[1][i] : w[0][i]);
      }
      turn_row(v, turn, p.interleaved);
      if (at.active && h < p.heads[side]) store_row<E>(p.y[side] + (here.t * p.heads[side] + h) * p.D, at, v);
      rows = next_rows;
      here = next;
    } while (here.piece == piece);
  }
}

// The weights' gradients are sums over all tokens: a wave keeps its own in registers over the tokens it takes, a workgroup adds
// its waves' and writes them, and the kernel below adds the workgroups' in order.  No atomics: the same bits every time.
template <class E, int G>
__global__ __launch_bounds__(64 * kNormWaves) void norm_rope_bwd_kernel(const NormRopeParams<E> p) {
  __shared__ float sums[kNormWaves][2][128];
  const int lane = threadIdx.x & 63, u = lane % G, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const RowPlace at = row_place(u, p.D, p.rotary, p.interleaved);
  const Walk<E, G, true> walk(p, at, lane);
  const int64_t stride = (int64_t)gridDim.x * kNormWaves;
  // (two steps ahead: with one, four waves to a SIMD hold 32 KiB to a compute unit in flight, and the kernel ran at 4.3 TB/s)
  auto advance = [&](const auto& w) __attribute__((always_inline)) {
    auto n = w;
    if (++n.step >= walk.steps) n = walk.first(w.piece + stride);
    return n;
  };
  auto here = walk.first((int64_t)blockIdx.x * kNormWaves + wave), next = advance(here);
  auto rows = walk.load(here), next_rows = walk.load(next);
  double position = walk.position(here), next_position = walk.position(next);
  const float inv_freq = 2 * lane < p.rotary ? p.inv_freq[lane] : 0.f;
  float w[2][8], dw[2][8] = {};
  load_weight(p, 0, at, w[0]);
  load_weight(p, 1, at, w[1]);
  const float over = 1.f / p.D;
  while (here.piece < walk.pieces) {
    const Turn turn = lane_turn(position, inv_freq, u, at.turned);
    const int64_t piece = here.piece;
    do {
      const auto after = advance(next);
      const auto after_rows = walk.load(after);
      const double after_position = after.piece != next.piece ? walk.position(after) : next_position;
      auto work = [&](auto side) __attribute__((always_inline)) {
        const int h = walk.head(here);
        const bool there = at.active && h < p.heads[side];
        float d[8];
        unpack<E>(rows.d, d);
        turn_row<true>(d, turn, p.interleaved);
        if (p.w[side]) {
          float v[8];
          unpack<E>(rows.x, v);
          float sq = 0.f, dot = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            sq += v[i] * v[i];
            dot += d[i] * w[side][i] * v[i];
          }
          const float r = 1.f / sqrtf(row_sum<G>(sq) * over + p.eps);
          const float m = row_sum<G>(dot) * r * over;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float n = v[i] * r;
            if (there) dw[side][i] += d[i] * n;
            d[i] = r * (d[i] * w[side][i] - n * m);
          }
        }
        if (there) store_row<E>(p.y[side] + (here.t * p.heads[side] + h) * p.D, at, d);
      };
      if (walk.side(here)) work(std::integral_constant<int, 1>{});
      else work(std::integral_constant<int, 0>{});
      rows = next_rows;
      here = next;
      position = next_position;
      next_rows = after_rows;
      next = after;
      next_position = after_position;
    } while (here.piece == piece);
  }
  if (!p.partials) return;
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int o = G; o < 64; o <<= 1) dw[side][i] += __shfl_xor(dw[side][i], o, 64);
      if (lane < G && at.active) sums[wave][side][(i < 4 ? at.a : at.b - 4) + i] = dw[side][i];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.D; i += 64 * kNormWaves) {
    const int side = i >= p.D, e = i - side * p.D;
    float s = 0.f;
    for (int v = 0; v < kNormWaves; ++v) s += sums[v][side][e];
    p.partials[(int64_t)blockIdx.x * 2 * p.D + i] = s;
  }
}

// dw[side][e] = sum of the workgroups' parts, 16 columns to a workgroup, 64 rows at a time; in 64 bits, rounded once
constexpr int kSumCols = 16, kSumRows = 64, kSumWaves = kSumCols * kSumRows / 64;
template <class E>
__global__ __launch_bounds__(kSumCols * kSumRows) void norm_rope_sum_kernel(const float* __restrict__ partials, int n, int D,
                                                                            void* dq_weight, void* dk_weight, int w32) {
  __shared__ double sums[kSumWaves][kSumCols];
  const int c = threadIdx.x % kSumCols, r = threadIdx.x / kSumCols, col = blockIdx.x * kSumCols + c;
  double s = 0.;
#pragma unroll 8
  for (int i = r; i < n; i += kSumRows) s += (double)partials[(int64_t)i * 2 * D + col];
  s += __shfl_xor(s, 16, 64);
  s += __shfl_xor(s, 32, 64);
  if ((threadIdx.x & 63) < kSumCols) sums[threadIdx.x >> 6][c] = s;
  __syncthreads();
  if (r != 0) return;
  s = 0.;
#pragma unroll
  for (int i = 0; i < kSumWaves; ++i) s += sums[i][c];
  void* dw = col < D ? dq_weight : dk_weight;
  const int e = col < D ? col : col - D;
  if (!dw) return;
  if (w32) ((float*)dw)[e] = (float)s;
  else ((typename E::elem*)dw)[e] = (typename E::elem)(float)s;
}

}  // namespace moba

using namespace moba;

// workgroups of the backward kernel: four to a compute unit (sixteen waves) hold enough loads in flight
static int bwd_workgroups(int64_t S) {
  const int64_t most = 4LL * (compute_units() > 0 ? compute_units() : 256), need = (S + kNormWaves - 1) / kNormWaves;
  return (int)(need < most ? need : most);
}

static int check_norm_rope(const void* q, const void* k, const void* yq, const void* yk, const void* positions,
                           const float* inv_freq, int64_t S, int H, int Hkv, int D, int rotary, const int64_t* strides,
                           int position_bits, int dtype) {
  if (!q || !k || !yq || !yk || !positions || !strides || (rotary > 0 && !inv_freq)) return MOBA_ERR_ARG;
  if (S <= 0 || H <= 0 || Hkv <= 0 || D <= 0 || (D & 7) || rotary < 0 || rotary > D || (rotary & 7)) return MOBA_ERR_ARG;
  if (position_bits != 32 && position_bits != 64) return MOBA_ERR_ARG;
  if (D > kHeadDim || (dtype != MOBA_DTYPE_BF16 && dtype != MOBA_DTYPE_F16)) return MOBA_ERR_UNSUPPORTED;
  for (const void* x : {q, k, yq, yk})
    if ((uintptr_t)x & 7) return MOBA_ERR_ARG;
  for (int i = 0; i < 4; ++i)
    if (strides[i] & 3) return MOBA_ERR_ARG;  // 8-byte accesses
  if (S > (1LL << 25) || H > (1 << 16) || Hkv > (1 << 16)) return MOBA_ERR_LIMIT;  // (threads of a launch: 32 bits)
  return MOBA_OK;
}

template <class E>
static NormRopeParams<E> norm_rope_params(const void* q, const void* k, void* yq, void* yk, const void* qw, const void* kw,
                                          const void* positions, const float* inv_freq, int64_t S, int H, int Hkv, int D,
                                          int rotary, const int64_t* strides, int position_bits, int interleaved, int w32,
                                          float eps) {
  typedef typename E::elem elem;
  NormRopeParams<E> p = {};
  p.x[0] = (const elem*)q; p.x[1] = (const elem*)k;
  p.y[0] = (elem*)yq; p.y[1] = (elem*)yk;
  p.w[0] = qw; p.w[1] = kw;
  p.positions = positions; p.inv_freq = inv_freq;
  p.S = S; p.heads[0] = H; p.heads[1] = Hkv; p.D = D; p.rotary = rotary;
  p.tok_stride[0] = strides[0]; p.head_stride[0] = strides[1];
  p.tok_stride[1] = strides[2]; p.head_stride[1] = strides[3];
  p.eps = eps; p.position64 = position_bits == 64; p.w32 = w32; p.interleaved = interleaved != 0;
  p.parts = 1;
  return p;
}

template <class E>
static int launch_norm_rope(NormRopeParams<E> p, hipStream_t st) {
  LaunchCheck launch_check;
  const int rows = p.D > 64 ? 4 : 8;
  // with few tokens, as many waves to a token as it has steps, up to sixteen waves to a compute unit
  const int most = (p.heads[0] + rows - 1) / rows + (p.heads[1] + rows - 1) / rows;
  const int cus = compute_units() > 0 ? compute_units() : 256;
  const int64_t want = (16LL * cus + p.S - 1) / p.S;
  p.parts = (int)(want < most ? want : most);
  // A wave for every token, but for up to a few tokens to each wave that the chip holds, where new waves cost more than they
  // balance: 20480 tokens, 10 heads: 27.7 us, 24.6 so; 131072 tokens, 40 heads: 489, 534 so
  const int64_t need = (p.S * p.parts + kNormWaves - 1) / kNormWaves, held = (int64_t)kNormResident * cus;
  const int64_t wgs = need > held && need <= 4 * held ? held : need;
  if (p.D > 64) hipLaunchKernelGGL((norm_rope_kernel<E, 16>), dim3((unsigned)wgs), dim3(64 * kNormWaves), 0, st, p);
  else hipLaunchKernelGGL((norm_rope_kernel<E, 8>), dim3((unsigned)wgs), dim3(64 * kNormWaves), 0, st, p);
  return launch_check.result();
}

extern "C" int moba_qk_norm_rope(const void* q, const void* k, void* yq, void* yk, const void* q_weight, const void* k_weight,
                                 const void* positions, const float* inv_freq, int64_t S, int H, int Hkv, int D, int rotary,
                                 const int64_t* strides, int position_bits, int interleaved, int weight_f32, float eps,
                                 int dtype, void* stream) {
  const int rc = check_norm_rope(q, k, yq, yk, positions, inv_freq, S, H, Hkv, D, rotary, strides, position_bits, dtype);
  if (rc != MOBA_OK) return rc;
  const uintptr_t w_align = weight_f32 ? 3 : 7;
  if (((uintptr_t)q_weight & w_align) || ((uintptr_t)k_weight & w_align)) return MOBA_ERR_ARG;
#define MOBA_NORM_ROPE(E)                                                                                                  \
  launch_norm_rope<E>(norm_rope_params<E>(q, k, yq, yk, q_weight, k_weight, positions, inv_freq, S, H, Hkv, D, rotary,      \
                                          strides, position_bits, interleaved, weight_f32, eps), (hipStream_t)stream)
  return dtype == MOBA_DTYPE_F16 ? MOBA_NORM_ROPE(F16) : MOBA_NORM_ROPE(Bf16);
#undef MOBA_NORM_ROPE
}

extern "C" size_t moba_qk_norm_rope_bwd_workspace_bytes(int64_t S, int D) {
  return S <= 0 || D <= 0 ? 0 : (size_t)bwd_workgroups(S) * 2 * D * sizeof(float);
}

template <class E>
static int launch_norm_rope_bwd(NormRopeParams<E> p, void* dqw, void* dkw, hipStream_t st) {
  LaunchCheck launch_check;
  const int wgs = bwd_workgroups(p.S);
  if (p.D > 64) hipLaunchKernelGGL((norm_rope_bwd_kernel<E, 16>), dim3(wgs), dim3(64 * kNormWaves), 0, st, p);
  else hipLaunchKernelGGL((norm_rope_bwd_kernel<E, 8>), dim3(wgs), dim3(64 * kNormWaves), 0, st, p);
  if (p.partials)
    hipLaunchKernelGGL(norm_rope_sum_kernel<E>, dim3(2 * p.D / kSumCols), dim3(kSumCols * kSumRows), 0, st,
                       (const float*)p.partials, wgs, p.D, dqw, dkw, p.w32);
  return launch_check.result();
}

extern "C" int moba_qk_norm_rope_bwd(const void* dyq, const void* dyk, const void* q, const void* k, void* dq, void* dk,
                                     const void* q_weight, const void* k_weight, void* dq_weight, void* dk_weight,
                                     void* workspace, const void* positions, const float* inv_freq, int64_t S, int H, int Hkv,
                                     int D, int rotary, const int64_t* strides, int position_bits, int interleaved,
                                     int weight_f32, float eps, int dtype, void* stream) {
  const int rc = check_norm_rope(q, k, dq, dk, positions, inv_freq, S, H, Hkv, D, rotary, strides, position_bits, dtype);
  if (rc != MOBA_OK) return rc;
  const uintptr_t w_align = weight_f32 ? 3 : 7;
  if (!dyq || !dyk || ((uintptr_t)dyq & 7) || ((uintptr_t)dyk & 7)) return MOBA_ERR_ARG;
  if (((uintptr_t)q_weight & w_align) || ((uintptr_t)k_weight & w_align)) return MOBA_ERR_ARG;
  const bool sums = dq_weight || dk_weight;
  if ((dq_weight && !q_weight) || (dk_weight && !k_weight) || (sums && (!workspace || ((uintptr_t)workspace & 3)))) return MOBA_ERR_ARG;
  if (((uintptr_t)dq_weight | (uintptr_t)dk_weight) & (weight_f32 ? 3 : 1)) return MOBA_ERR_ARG;
#define MOBA_NORM_ROPE_BWD(E)                                                                                               \
  {                                                                                                                         \
    NormRopeParams<E> p = norm_rope_params<E>(q, k, dq, dk, q_weight, k_weight, positions, inv_freq, S, H, Hkv, D, rotary,  \
                                              strides, position_bits, interleaved, weight_f32, eps);                        \
    p.dy[0] = (const E::elem*)dyq;                                                                                          \
    p.dy[1] = (const E::elem*)dyk;                                                                                          \
    p.partials = sums ? (float*)workspace : nullptr;                                                                        \
    return launch_norm_rope_bwd<E>(p, dq_weight, dk_weight, (hipStream_t)stream);                                           \
  }
  if (dtype == MOBA_DTYPE_F16) MOBA_NORM_ROPE_BWD(F16)
  MOBA_NORM_ROPE_BWD(Bf16)
#undef MOBA_NORM_ROPE_BWD
}
