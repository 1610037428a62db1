// Products with 4-bit weights and the experts' feed-forward networks (oracle/decode_engine.py:122-133).
//
//   linear:   y[t, n] = sum_k x[t, k] W[n, k]
//   experts:  y[t] = sum_j down_e( w_tj silu(min(g, lim)) clamp(u, -lim, lim) ),  g = gate_e x_t, u = up_e x_t,
//             e = ids[t, j]; an id outside 0 .. E-1 adds nothing.
//
// Products run on the bf16 matrix cores with fp32 sums; the weights are e2m1 codes (fp4.h) or bf16.  The hidden
// row, its router weight in it, is rounded to bf16 once: it is an operand of the second product, and half a step of
// its 8 bits is what y's own rounding costs again.
#include "fp4.h"
#include "smla_internal.h"

namespace {

using smla_fp4::scale_of;
using smla_fp4::to_bf16;

constexpr int kFp4 = 0, kBf16 = 1;

// A matrix of rows of K weights: codes (K / 2 bytes a row) and scale bytes (K / 32), or bf16.
struct Matrix {
  const uint8_t* w;
  const uint8_t* s;
};

// 32 weights of a row, and their 8 values j = 0 .. 3
template <int WT>
struct Block;
template <>
struct Block<kFp4> {
  u32x4_t c;
  uint32_t s;
  __device__ void load(const Matrix& m, int64_t row, int K, int kb) {
    c = *(const u32x4_t*)(m.w + row * (K / 2) + 16 * kb);
    s = m.s[row * (K / 32) + kb];
  }
  __device__ void zero() { c = u32x4_t{0, 0, 0, 0}, s = 127; }
  __device__ bf16x8_t frag(int j) const { return to_bf16(c[j], scale_of(s)); }
};
template <>
struct Block<kBf16> {
  u32x4_t c[4];
  __device__ void load(const Matrix& m, int64_t row, int K, int kb) {
    const uint8_t* p = m.w + (row * K + 32 * kb) * 2;
#pragma unroll
    for (int j = 0; j < 4; j++) c[j] = *(const u32x4_t*)(p + 16 * j);
  }
  __device__ void zero() {
#pragma unroll
    for (int j = 0; j < 4; j++) c[j] = u32x4_t{0, 0, 0, 0};
  }
  __device__ bf16x8_t frag(int j) const { return as_bf16x8(c[j]); }
};

constexpr int kWaves = 8;

// acc[r] (rows 16 r + 4 q .. +3 of the tile, column m of lane 16 q + m) += the wave's share of the K range, for R
// matrices' rows; x: this lane's column, null where there is none.  A step is 128 k: lane group q takes the 32 of
// block 4 s + q on both sides.
template <int WT, int R>
__device__ inline void products(const Matrix (&m)[R], const int64_t (&row)[R], const uint16_t* x, int K, f32x4_t (&acc)[R]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
  const int nb = K / 32, steps = (nb + 3) / 4;
  const int s0 = steps * wave / kWaves, s1 = steps * (wave + 1) / kWaves;
#pragma unroll
  for (int r = 0; r < R; r++) acc[r] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int s = s0; s < s1; s++) {
    const int kb = 4 * s + q;
    Block<WT> w[R];
    u32x4_t xv[4];
#pragma unroll
    for (int j = 0; j < 4; j++) xv[j] = u32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int r = 0; r < R; r++) w[r].zero();
    if (kb < nb) {
#pragma unroll
      for (int r = 0; r < R; r++) w[r].load(m[r], row[r], K, kb);
      if (x) {
#pragma unroll
        for (int j = 0; j < 4; j++) xv[j] = *(const u32x4_t*)(x + 32 * kb + 8 * j);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int r = 0; r < R; r++)
        acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[r].frag(j), as_bf16x8(xv[j]), acc[r], 0, 0, 0);
  }
}

// the waves' sums, in wave order, in wave 0
template <int R>
__device__ inline void join(f32x4_t (&acc)[R]) {
  __shared__ f32x4_t red[kWaves][R][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int r = 0; r < R; r++) red[wave][r][lane] = acc[r];
  __syncthreads();
  if (wave != 0) return;
  for (int v = 1; v < kWaves; v++)
#pragma unroll
    for (int r = 0; r < R; r++) {
      const f32x4_t p = red[v][r][lane];
#pragma unroll
      for (int i = 0; i < 4; i++) acc[r][i] += p[i];
    }
}

template <int YDT>
__device__ inline void store4(void* y, int64_t at, int n, int N, const f32x4_t& v) {
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (n + i < N) {
      if constexpr (YDT == SMLA_BF16) ((uint16_t*)y)[at + i] = bf16_rne(v[i]);
      else ((float*)y)[at + i] = v[i];
    }
}

template <int YDT>
__global__ __launch_bounds__(64 * kWaves) void linear_fp4_kernel(const uint16_t* __restrict__ x, int64_t ldx, Matrix w, int T,
                                                                 int N, int K, void* __restrict__ y) {
  const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16, t = blockIdx.y * 16 + m;
  f32x4_t acc[1];
  products<kFp4, 1>({w}, {(int64_t)min(n0 + m, N - 1)}, t < T ? x + (int64_t)t * ldx : nullptr, K, acc);
  join(acc);
  if (threadIdx.x < 64 && t < T) store4<YDT>(y, (int64_t)t * N + n0 + 4 * q, n0 + 4 * q, N, acc[0]);
}

// ---- the experts

struct ExpertArgs {
  const uint16_t* x;
  int64_t ldx;
  const int32_t* ids;
  const float* weights;
  int T, k, E, K, I, P;  // P = T k pairs
  Matrix gate, up, down;
  float limit;           // infinity: none
  int32_t* list;         // pairs by expert
  int32_t* tiles;        // [0] their number, then (expert, first pair, pairs) each
  uint16_t* h;           // [P, I] hidden rows, by pair
  float* part;           // [P, K]
  uint16_t* y;
};

constexpr int kMaxExperts = 1024, kTile = 16;

// The pairs (token, place) by expert, and tiles of up to kTile of an expert's.  The order within an expert is as
// it comes; no result depends on it.
__global__ __launch_bounds__(1024) void plan_kernel(const ExpertArgs a) {
  __shared__ int cnt[kMaxExperts], at[kMaxExperts], tile[kMaxExperts];
  const int tid = threadIdx.x;
  cnt[tid] = 0;
  __syncthreads();
  for (int p = tid; p < a.P; p += 1024) {
    const int e = a.ids[p];
    if (e >= 0 && e < a.E) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  const int n = cnt[tid], nt = (n + kTile - 1) / kTile;
  at[tid] = n, tile[tid] = nt;
  __syncthreads();
  for (int o = 1; o < 1024; o *= 2) {  // inclusive sums
    const int u = tid >= o ? at[tid - o] : 0, v = tid >= o ? tile[tid - o] : 0;
    __syncthreads();
    at[tid] += u, tile[tid] += v;
    __syncthreads();
  }
  const int first = at[tid] - n, t0 = tile[tid] - nt;
  if (tid == 1023) a.tiles[0] = tile[tid];
  for (int i = 0; i < nt; i++) {
    a.tiles[1 + 3 * (t0 + i)] = tid;
    a.tiles[2 + 3 * (t0 + i)] = first + i * kTile;
    a.tiles[3 + 3 * (t0 + i)] = min(kTile, n - i * kTile);
  }
  __syncthreads();
  at[tid] = first;
  __syncthreads();
  for (int p = tid; p < a.P; p += 1024) {
    const int e = a.ids[p];
    if (e >= 0 && e < a.E) a.list[atomicAdd(&at[e], 1)] = p;
  }
}

__device__ inline float gated(float g, float u, float lim) {
  g = fminf(g, lim), u = fminf(fmaxf(u, -lim), lim);
  return g / (1.f + __expf(-g)) * u;
}

template <int WT>
__global__ __launch_bounds__(64 * kWaves) void up_kernel(const ExpertArgs a) {
  if ((int)blockIdx.y >= a.tiles[0]) return;
  const int* tl = a.tiles + 1 + 3 * blockIdx.y;
  const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4, e = tl[0];
  const int p = m < tl[2] ? a.list[tl[1] + m] : -1, i0 = blockIdx.x * 16;
  const int64_t row = (int64_t)e * a.I + i0 + m;
  f32x4_t acc[2];
  products<WT, 2>({a.gate, a.up}, {row, row}, p >= 0 ? a.x + (int64_t)(p / a.k) * a.ldx : nullptr, a.K, acc);
  join(acc);
  if (threadIdx.x < 64 && p >= 0) {
    const float w = a.weights[p];
    f32x4_t h;
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = w * gated(acc[0][i], acc[1][i], a.limit);
    store4<SMLA_BF16>(a.h, (int64_t)p * a.I + i0 + 4 * q, 0, 4, h);
  }
}

template <int WT>
__global__ __launch_bounds__(64 * kWaves) void down_kernel(const ExpertArgs a) {
  if ((int)blockIdx.y >= a.tiles[0]) return;
  const int* tl = a.tiles + 1 + 3 * blockIdx.y;
  const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4, e = tl[0];
  const int p = m < tl[2] ? a.list[tl[1] + m] : -1, n0 = blockIdx.x * 16;
  f32x4_t acc[1];
  products<WT, 1>({a.down}, {(int64_t)e * a.K + n0 + m}, p >= 0 ? a.h + (int64_t)p * a.I : nullptr, a.I, acc);
  join(acc);
  if (threadIdx.x < 64 && p >= 0) store4<SMLA_F32>(a.part, (int64_t)p * a.K + n0 + 4 * q, 0, 4, acc[0]);
}

// y[t] = the sum of its pairs' rows, in their order
__global__ __launch_bounds__(256) void combine_kernel(const ExpertArgs a) {
  const int t = blockIdx.y, n = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (n >= a.K) return;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < a.k; j++) {
    const int p = t * a.k + j, e = a.ids[p];
    if (e >= 0 && e < a.E) sum += *(const f32x4_t*)(a.part + (int64_t)p * a.K + n);
  }
  *(u32x2_t*)(a.y + (int64_t)t * a.K + n) = u32x2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
}

int64_t up16(int64_t n) { return (n + 15) & ~(int64_t)15; }
int64_t max_tiles(int64_t P, int64_t E) { return P / kTile + (E < P ? E : P); }

int check_experts(int64_t T, int64_t k, int64_t E, int64_t K, int64_t I) {
  if (T <= 0 || k <= 0 || E <= 0 || K <= 0 || I <= 0) return SMLA_E_SHAPE;
  if (K % 32 != 0 || I % 32 != 0 || E > kMaxExperts || k > 64 || K > (1 << 20) || I > (1 << 20) || T > 65535) return SMLA_E_UNSUPPORTED;
  return SMLA_OK;
}

template <int WT>
int launch_experts(const ExpertArgs& a, hipStream_t st) {
  const unsigned nt = (unsigned)max_tiles(a.P, a.E);
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(1024), 0, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  hipLaunchKernelGGL(up_kernel<WT>, dim3(a.I / 16, nt), dim3(64 * kWaves), 0, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  hipLaunchKernelGGL(down_kernel<WT>, dim3(a.K / 16, nt), dim3(64 * kWaves), 0, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  hipLaunchKernelGGL(combine_kernel, dim3((a.K / 4 + 255) / 256, a.T), dim3(256), 0, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

}  // namespace

extern "C" size_t smla_linear_fp4_workspace(int64_t T, int64_t N, int64_t K) {
  (void)T, (void)N, (void)K;
  return 0;
}

extern "C" int smla_linear_fp4(const void* x, int64_t ldx, const uint8_t* codes, const uint8_t* scales, int64_t T, int64_t N,
                               int64_t K, void* y, int y_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  (void)workspace, (void)workspace_bytes;
  if (T < 0 || N <= 0 || K <= 0 || (T > 1 && ldx < K)) return SMLA_E_SHAPE;
  if (y_dtype != SMLA_BF16 && y_dtype != SMLA_F32) return SMLA_E_DTYPE;
  if (T == 0) return SMLA_OK;
  if (!x || !codes || !scales || !y) return SMLA_E_NULL;
  if (K % 32 != 0 || ldx % 8 != 0 || ((uintptr_t)x & 15) || ((uintptr_t)codes & 15) || T > 65535 * 16 || N > (1 << 24) || K > (1 << 24))
    return SMLA_E_UNSUPPORTED;
  const dim3 grid((unsigned)((N + 15) / 16), (unsigned)((T + 15) / 16)), blk(64 * kWaves);
  auto kern = y_dtype == SMLA_BF16 ? linear_fp4_kernel<SMLA_BF16> : linear_fp4_kernel<SMLA_F32>;
  hipLaunchKernelGGL(kern, grid, blk, 0, (hipStream_t)stream, (const uint16_t*)x, ldx, Matrix{codes, scales}, (int)T, (int)N, (int)K, y);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

extern "C" size_t smla_experts_workspace(int64_t T, int64_t k, int64_t E, int64_t K, int64_t I) {
  if (check_experts(T, k, E, K, I) != SMLA_OK) return 0;
  const int64_t P = T * k;
  return (size_t)(up16(4 * P) + up16(4 + 12 * max_tiles(P, E)) + up16(2 * P * I) + 4 * P * K);
}

extern "C" int smla_experts(const void* x, int64_t ldx, const int32_t* ids, const float* weights, int64_t T, int64_t k, int64_t E,
                            int64_t K, int64_t I, const void* gate, const uint8_t* gate_scales, const void* up,
                            const uint8_t* up_scales, const void* down, const uint8_t* down_scales, int w_dtype, float limit,
                            void* y, void* workspace, size_t workspace_bytes, void* stream) {
  if (w_dtype != SMLA_BF16 && w_dtype != SMLA_FP4_E2M1) return SMLA_E_DTYPE;
  if (T == 0 && k > 0 && E > 0 && K > 0 && I > 0) return SMLA_OK;
  int rc = check_experts(T, k, E, K, I);
  if (rc) return rc;
  const bool fp4 = w_dtype == SMLA_FP4_E2M1;
  if (!x || !ids || !weights || !gate || !up || !down || !y || (fp4 && (!gate_scales || !up_scales || !down_scales))) return SMLA_E_NULL;
  if (T > 1 && ldx < K) return SMLA_E_SHAPE;
  if (!(limit > 0.f)) return SMLA_E_RANGE;
  if (ldx % 8 != 0 || (((uintptr_t)x | (uintptr_t)gate | (uintptr_t)up | (uintptr_t)down | (uintptr_t)y) & 15)) return SMLA_E_UNSUPPORTED;
  if (!usable_workspace(workspace, workspace_bytes, smla_experts_workspace(T, k, E, K, I))) return SMLA_E_WORKSPACE;
  const int64_t P = T * k;
  ExpertArgs a{(const uint16_t*)x, ldx, ids, weights, (int)T, (int)k, (int)E, (int)K, (int)I, (int)P,
               {(const uint8_t*)gate, gate_scales}, {(const uint8_t*)up, up_scales}, {(const uint8_t*)down, down_scales}, limit,
               nullptr, nullptr, nullptr, nullptr, (uint16_t*)y};
  uint8_t* ws = (uint8_t*)workspace;
  a.list = (int32_t*)ws, ws += up16(4 * P);
  a.tiles = (int32_t*)ws, ws += up16(4 + 12 * max_tiles(P, E));
  a.h = (uint16_t*)ws, ws += up16(2 * P * I);
  a.part = (float*)ws;
  return fp4 ? launch_experts<kFp4>(a, (hipStream_t)stream) : launch_experts<kBf16>(a, (hipStream_t)stream);
}
