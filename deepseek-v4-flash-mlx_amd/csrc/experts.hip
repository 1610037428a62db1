// Products with 4-bit weights and the experts' feed-forward networks (oracle/decode_engine.py:122-133).
//
//   linear:   y[t, n] = sum_k x[t, k] W[n, k]
//   experts:  y[t] = sum_j down_e( w_tj silu(min(g, lim)) clamp(u, -lim, lim) ),  g = gate_e x_t, u = up_e x_t,
//             e = ids[t, j]; an id outside 0 .. E-1 adds nothing.
//
// Products run on the bf16 matrix cores with fp32 sums; the weights are e2m1 codes (fp4.h) or bf16.  The hidden
// row, its router weight in it, is rounded to bf16 once: it is an operand of the second product, and half a step of
// its 8 bits is what y's own rounding costs again.
#include "expert_tile.h"
#include "fp4.h"
#include "smla_internal.h"

namespace {

using smla_fp4::scale_of;
using smla_fp4::to_bf16;
using smla_tile::kBf16;
using smla_tile::kFp4;

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

// ---- few tokens (up to 16): the weights are streamed once, a 16-row block of W (A of the product) against all tokens
// (B: column m of lane 16 q + m is token m).  A step is 128 k: lane group q takes the 32 of block 4 s + q on both
// sides, 16 bytes of codes a lane.  The K range is cut over the waves of a workgroup, kAhead steps' loads are in flight.

constexpr int kFew = 16;
template <int WT>
constexpr int kAhead = WT == kFp4 ? 4 : 2;

__device__ inline void add4(f32x4_t& a, const f32x4_t& b) {
#pragma unroll
  for (int i = 0; i < 4; i++) a[i] += b[i];
}

// acc[r] (rows 4 q .. +3 of matrix r's 16, column m) = the sums over steps s0 .. s1-1 for R matrices' rows; x: this
// lane's column, null where there is none.
template <int WT, int R>
__device__ inline void products(const Matrix (&m)[R], int64_t row, const uint16_t* x, int K, int s0, int s1, f32x4_t (&acc)[R]) {
  constexpr int U = kAhead<WT>;
  const int q = (threadIdx.x >> 4) & 3, nb = K / 32;
#pragma unroll
  for (int r = 0; r < R; r++) acc[r] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  for (int s = s0; s < s1; s += U) {
    Block<WT> w[U][R];
    u32x4_t xv[U][4];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int kb = 4 * (s + u) + q;
#pragma unroll
      for (int r = 0; r < R; r++) w[u][r].zero();
#pragma unroll
      for (int j = 0; j < 4; j++) xv[u][j] = u32x4_t{0, 0, 0, 0};
      if (s + u < s1 && kb < nb) {
#pragma unroll
        for (int r = 0; r < R; r++) w[u][r].load(m[r], row, K, kb);
        if (x) {
#pragma unroll
          for (int j = 0; j < 4; j++) xv[u][j] = *(const u32x4_t*)(x + 32 * kb + 8 * j);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int r = 0; r < R; r++)
          acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[u][r].frag(j), as_bf16x8(xv[u][j]), acc[r], 0, 0, 0);
  }
}

// the waves' sums, in wave order, in wave 0
template <int NW, int R>
__device__ inline void join(f32x4_t (&acc)[R]) {
  __shared__ f32x4_t red[NW][R][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int r = 0; r < R; r++) red[wave][r][lane] = acc[r];
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int v = 1; v < NW; v++)
#pragma unroll
    for (int r = 0; r < R; r++) add4(acc[r], red[v][r][lane]);
}

template <int NW, int YDT>
__global__ __launch_bounds__(64 * NW) void linear_few_kernel(const uint16_t* __restrict__ x, int64_t ldx, Matrix w, int T, int N,
                                                             int K, void* __restrict__ y) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, q = lane >> 4, steps = (K + 127) / 128;
  const int n0 = blockIdx.x * 16;
  f32x4_t acc[1];
  products<kFp4, 1>({w}, min(n0 + m, N - 1), m < T ? x + (int64_t)m * ldx : nullptr, K, steps * wave / NW, steps * (wave + 1) / NW, acc);
  join<NW>(acc);
  if (wave != 0 || m >= T) return;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int n = n0 + 4 * q + i;
    if (n < N) {
      if constexpr (YDT == SMLA_BF16) ((uint16_t*)y)[(int64_t)m * N + n] = bf16_rne(acc[0][i]);
      else ((float*)y)[(int64_t)m * N + n] = acc[0][i];
    }
  }
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
  int32_t* at;           // a pair's place in it
  int32_t* tiles;        // [0] their number, then (expert, first place, pairs) each
  int tile;              // pairs of a tile at most
  uint16_t* h;           // [P, I] hidden rows, by place (few tokens: by pair)
  float* part;           // [P, K] their products, by place
  uint16_t* y;
};

constexpr int kMaxExperts = 1024, kMaxChoices = 64;

__device__ inline float gated(float g, float u, float lim) {
  g = fminf(g, lim), u = fminf(fmaxf(u, -lim), lim);
  return g / (1.f + __expf(-g)) * u;
}

// Workgroup (i, p): 16 hidden rows' gate and up products of the expert of pair p, where p is its first pair, for
// every token that has it.  A token that has it twice has the sum of its weights.
constexpr int kUpWaves = 8;
template <int WT>
__global__ __launch_bounds__(64 * kUpWaves) void few_up_kernel(const ExpertArgs a) {
  const int p = blockIdx.y, e = a.ids[p], lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, q = lane >> 4;
  if (e < 0 || e >= a.E) return;
  bool seen = false;
  for (int o = lane; o < p; o += 64) seen |= a.ids[o] == e;
  if (__any(seen)) return;
  int pair = -1;
  float w = 0.f;
  if (m < a.T)
    for (int j = a.k - 1; j >= 0; j--)
      if (a.ids[m * a.k + j] == e) pair = m * a.k + j, w += a.weights[pair];
  const int i0 = blockIdx.x * 16, steps = (a.K + 127) / 128;
  f32x4_t acc[2];
  products<WT, 2>({a.gate, a.up}, (int64_t)e * a.I + i0 + m, pair >= 0 ? a.x + m * a.ldx : nullptr, a.K, steps * wave / kUpWaves,
                  steps * (wave + 1) / kUpWaves, acc);
  join<kUpWaves>(acc);
  if (wave != 0 || pair < 0) return;
  float h[4];
#pragma unroll
  for (int i = 0; i < 4; i++) h[i] = w * gated(acc[0][i], acc[1][i], a.limit);
  *(u32x2_t*)(a.h + (int64_t)pair * a.I + i0 + 4 * q) = u32x2_t{pack_bf16x2(h[0], h[1]), pack_bf16x2(h[2], h[3])};
}

// Workgroup i: 16 columns of y for every token, over all experts that any token has: the waves share out the K
// ranges of all of them.  A wave adds an expert's sums to a token's only where the token has it (0 times an infinite
// weight of another token's expert would be NaN).
constexpr int kDownWaves = 16;
template <int WT>
__global__ __launch_bounds__(64 * kDownWaves) void few_down_kernel(const ExpertArgs a) {
  constexpr int U = kAhead<WT>;
  __shared__ int32_t ids[kFew * kMaxChoices], act[kFew * kMaxChoices];
  __shared__ int16_t pairs[kFew * kMaxChoices][kFew];
  __shared__ int cnt[kDownWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, q = lane >> 4;
  const int e0 = tid < a.P ? a.ids[tid] : -1;
  ids[tid] = e0;
  __syncthreads();
  bool first = e0 >= 0 && e0 < a.E;
  for (int o = 0; first && o < tid; o++) first = ids[o] != e0;
  const uint64_t mask = __ballot(first);
  if (lane == 0) cnt[wave] = __popcll(mask);
  __syncthreads();
  int at = 0, n = 0;
  for (int v = 0; v < kDownWaves; v++) {
    if (v < wave) at += cnt[v];
    n += cnt[v];
  }
  if (first) act[at + __popcll(mask & ((1ull << lane) - 1))] = e0;
  __syncthreads();
  for (int i = tid; i < n * kFew; i += 64 * kDownWaves) {
    const int t = i % kFew, e = act[i / kFew];
    int pair = -1;
    if (t < a.T)
      for (int j = a.k - 1; j >= 0; j--)
        if (ids[t * a.k + j] == e) pair = t * a.k + j;
    pairs[i / kFew][t] = (int16_t)pair;
  }
  __syncthreads();
  const int n0 = blockIdx.x * 16, nb = a.I / 32, per = (nb + 3) / 4, steps = n * per;
  const int s0 = steps * wave / kDownWaves, s1 = steps * (wave + 1) / kDownWaves;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f}, acc = sum;
  int cur = s0 / per, k0 = s0 - cur * per;  // expert and its step, of the loads
  int has = -1, of = cur;
  if (s0 < s1) has = pairs[cur][m];
  for (int s = s0; s < s1; s += U) {
    Block<WT> w[U];
    u32x4_t xv[U][4];
    int ex[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int kb = 4 * k0 + q;
      ex[u] = cur;
      w[u].zero();
#pragma unroll
      for (int j = 0; j < 4; j++) xv[u][j] = u32x4_t{0, 0, 0, 0};
      if (s + u < s1) {
        if (kb < nb) {
          w[u].load(a.down, (int64_t)act[cur] * a.K + n0 + m, a.I, kb);
          const int pair = pairs[cur][m];
          if (pair >= 0) {
#pragma unroll
            for (int j = 0; j < 4; j++) xv[u][j] = *(const u32x4_t*)(a.h + (int64_t)pair * a.I + 32 * kb + 8 * j);
          }
        }
        if (++k0 == per) k0 = 0, cur++;
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (s + u >= s1) break;
      if (ex[u] != of) {
        if (has >= 0) add4(sum, acc);
        acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
        of = ex[u];
        has = pairs[of][m];
      }
#pragma unroll
      for (int j = 0; j < 4; j++) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[u].frag(j), as_bf16x8(xv[u][j]), acc, 0, 0, 0);
    }
  }
  if (has >= 0) add4(sum, acc);
  f32x4_t all[1] = {sum};
  join<kDownWaves>(all);
  if (wave != 0 || m >= a.T) return;
  *(u32x2_t*)(a.y + (int64_t)m * a.K + n0 + 4 * q) = u32x2_t{pack_bf16x2(all[0][0], all[0][1]), pack_bf16x2(all[0][2], all[0][3])};
}

// ---- more tokens: the pairs (token, choice) sorted by expert, in tiles of one expert's.  The order within an expert is
// as it comes; no result depends on it.
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
  const int n = cnt[tid], nt = (n + a.tile - 1) / a.tile;
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
    a.tiles[2 + 3 * (t0 + i)] = first + i * a.tile;
    a.tiles[3 + 3 * (t0 + i)] = min(a.tile, n - i * a.tile);
  }
  __syncthreads();
  at[tid] = first;
  __syncthreads();
  for (int p = tid; p < a.P; p += 1024) {
    const int e = a.ids[p];
    if (e >= 0 && e < a.E) {
      const int i = atomicAdd(&at[e], 1);
      a.list[i] = p;
      a.at[p] = i;
    } else {
      a.at[p] = -1;
    }
  }
}

// y[t] = the sum of its pairs' rows, in their order
__global__ __launch_bounds__(256) void combine_kernel(const ExpertArgs a) {
  const int t = blockIdx.y, n = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (n >= a.K) return;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < a.k; j++) {
    const int i = a.at[(int64_t)t * a.k + j];
    if (i >= 0) add4(sum, *(const f32x4_t*)(a.part + (int64_t)i * a.K + n));
  }
  *(u32x2_t*)(a.y + (int64_t)t * a.K + n) = u32x2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
}

// Scale rows of whole steps: byte j of a row is scale j - lead of the source's row of nb, 127 (1) before it.
__global__ __launch_bounds__(256) void pad_scales_kernel(const uint8_t* __restrict__ s, int64_t rows, int nb, int ld,
                                                         uint8_t* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // four bytes
  if (i >= rows * (ld / 4)) return;
  const int64_t row = i / (ld / 4);
  const int j = (int)(i - row * (ld / 4)) * 4 - (ld - nb);
  uint32_t v = 0;
#pragma unroll
  for (int b = 0; b < 4; b++) v |= (j + b >= 0 ? (uint32_t)s[row * nb + j + b] : 127u) << (8 * b);
  ((uint32_t*)out)[i] = v;
}

// y[i] = the splits' sums, in their order
template <int YDT>
__global__ __launch_bounds__(256) void reduce_kernel(const float* __restrict__ part, int splits, int64_t n, void* __restrict__ y) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const int m = (int)min((int64_t)4, n - i);
  if (m == 4 && n % 4 == 0) {
    f32x4_t sum = *(const f32x4_t*)(part + i);
    for (int s = 1; s < splits; s++) add4(sum, *(const f32x4_t*)(part + s * n + i));
    if constexpr (YDT == SMLA_F32) *(f32x4_t*)((float*)y + i) = sum;
    else *(u32x2_t*)((uint16_t*)y + i) = u32x2_t{pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3])};
    return;
  }
  for (int e = 0; e < m; e++) {
    float sum = part[i + e];
    for (int s = 1; s < splits; s++) sum += part[s * n + i + e];
    if constexpr (YDT == SMLA_F32) ((float*)y)[i + e] = sum;
    else ((uint16_t*)y)[i + e] = bf16_rne(sum);
  }
}

// ---- tiles (expert_tile.h)

// tokens x outputs: waves of .. x .., stages
template <int WT, int FORM>
struct Form;
template <>
struct Form<kFp4, 0> : smla_tile::Tile<kFp4, 32, 256, 32, 64, 3> {};  // 75 KB, 4 waves: two workgroups a CU
template <>
struct Form<kFp4, 1> : smla_tile::Tile<kFp4, 64, 128, 32, 64, 3> {};  // 74 KB, 4 waves
template <>
struct Form<kFp4, 2> : smla_tile::Tile<kFp4, 128, 256, 64, 64, 3> {};  // 147 KB, 8 waves
template <>
struct Form<kFp4, 3> : smla_tile::Tile<kFp4, 128, 512, 64, 128, 2> {};  // 132 KB, 8 waves
template <>
struct Form<kBf16, 0> : smla_tile::Tile<kBf16, 32, 256, 32, 64, 4> {};  // 144 KB, 4 waves
template <>
struct Form<kBf16, 1> : smla_tile::Tile<kBf16, 64, 128, 32, 64, 3> {};  // 72 KB, 4 waves
template <>
struct Form<kBf16, 2> : smla_tile::Tile<kBf16, 128, 256, 64, 64, 3> {};  // 144 KB, 8 waves
constexpr int kFormBM[4] = {32, 64, 128, 128}, kFormBN[4] = {256, 128, 256, 512};

constexpr int kLinear = 0, kUp = 1, kDown = 2;

struct TileArgs {
  const uint8_t* x;
  int64_t ldx;          // bytes
  Matrix w[2];
  int64_t lds;          // bytes of a row of scales (a multiple of 4)
  int K, N;             // N: columns of the result
  int T;                // kLinear: tokens
  int nt, nn, splits;   // kLinear
  uint8_t* y;
  int64_t ldy, split_stride;  // elements
  int vec;
  // kUp, kDown
  const int32_t* tiles;
  const int32_t* list;
  const float* weights;
  int k;
  float limit;
};

template <class L, int MODE, int YDT, int MBV>
__device__ __attribute__((always_inline)) inline void tile_body(const TileArgs& a, smla_attn::lds_u8_t* lds, const smla_tile::Source& src,
                                                                int nk, int rows, int n0, uint8_t* y,
                                                                const smla_attn::lds_i32_t* tok, const smla_attn::lds_f32_t* wt) {
  f32x16_t acc[MBV > 0 ? MBV : 1][L::NB];
  constexpr int HALF = L::WN / 2;
  const int nmax = a.N - 1 - n0;
  smla_tile::tile_loop<L, MBV>(
      lds, src, nk,
      [&](int r) __attribute__((always_inline)) {
        if constexpr (MODE == kUp) return (uint32_t)tok[r] * (uint32_t)a.ldx;
        else return (uint32_t)min(r, rows - 1) * (uint32_t)a.ldx;
      },
      [&](int r) __attribute__((always_inline)) {
        if constexpr (MODE == kUp) return min(r / L::WN * HALF + r % HALF, nmax);
        else return min(r, nmax);
      },
      [&](int r) __attribute__((always_inline)) { return MODE == kUp ? r % L::WN / HALF : 0; }, acc);
  auto row = [&](int r) __attribute__((always_inline)) { return r < rows ? y + (int64_t)r * a.ldy * (YDT == SMLA_BF16 ? 2 : 4) : nullptr; };
  if constexpr (MODE == kUp) {
    const int lane = threadIdx.x & 63, wm = (threadIdx.x >> 6) / L::NWN;
    smla_tile::store_rows<L, MBV, L::NB / 2, YDT>(lds, a.vec, n0, a.N, [&](int m, int n, int r) __attribute__((always_inline)) {
      return wt[L::WM * wm + 32 * m + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)] * gated(acc[m][n][r], acc[m][n + L::NB / 2][r], a.limit);
    }, row);
  } else {
    smla_tile::store_rows<L, MBV, L::NB, YDT>(lds, a.vec, n0, a.N, [&](int m, int n, int r) __attribute__((always_inline)) { return acc[m][n][r]; },
                                             row);
  }
}

template <class L, int MODE, int YDT>
__global__ __launch_bounds__(L::THREADS) void tile_kernel(const TileArgs a) {
  extern __shared__ __align__(16) uint8_t lds_t[];
  smla_attn::lds_u8_t* lds = (smla_attn::lds_u8_t*)lds_t;
  smla_attn::lds_i32_t* tok = (smla_attn::lds_i32_t*)(lds + L::LDS);
  smla_attn::lds_f32_t* wt = (smla_attn::lds_f32_t*)(lds + L::LDS + 4 * L::BM);
  constexpr int BNO = MODE == kUp ? L::BN / 2 : L::BN;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), steps = (a.K + L::KB - 1) / L::KB, pad = steps * L::KB - a.K;
  int rows, n0, e = 0, s0 = 0, nk = steps;
  int64_t first;  // the tile's first row of x and y
  if constexpr (MODE == kLinear) {
    uint32_t id = smla_tile::xcd_run(gridDim.x);
    const uint32_t tiles = (uint32_t)a.nt * a.nn, sp = id / tiles;
    id -= sp * tiles;
    const uint32_t blk = 4u * a.nn, grp = id / blk, gs = min(4u, (uint32_t)a.nt - 4 * grp), in = id - grp * blk;
    first = (int64_t)(4 * grp + in % gs) * L::BM;
    n0 = in / gs * L::BN;
    rows = min((int64_t)L::BM, a.T - first);
    s0 = steps * sp / a.splits;
    nk = steps * (sp + 1) / a.splits - s0;
    const smla_tile::Source src{a.x + first * a.ldx + (int64_t)s0 * L::XROW - 2 * pad,
                                {a.w[0].w + (int64_t)n0 * (a.K * L::WROW / L::KB) + (int64_t)s0 * L::WROW - pad * L::WROW / L::KB, nullptr},
                                {a.w[0].s + (int64_t)n0 * a.lds + 4 * s0, nullptr},
                                (uint32_t)(a.K * L::WROW / L::KB), (uint32_t)a.lds, s0 == 0 ? pad : 0};
    uint8_t* y = a.y + (sp * a.split_stride + first * a.ldy) * (YDT == SMLA_BF16 ? 2 : 4);
    const int mine = rows - L::WM * (wave / L::NWN);
    if (mine > 32 * (L::MB - 1)) tile_body<L, MODE, YDT, L::MB>(a, lds, src, nk, rows, n0, y, tok, wt);
    else if (mine <= 0) tile_body<L, MODE, YDT, 0>(a, lds, src, nk, rows, n0, y, tok, wt);
    else if constexpr (L::MB == 2) tile_body<L, MODE, YDT, 1>(a, lds, src, nk, rows, n0, y, tok, wt);
  } else {
    const uint32_t ntn = (a.N + BNO - 1) / BNO, tot = a.tiles[0] * ntn, id = smla_tile::xcd_run(tot);
    if (id >= tot) return;
    const uint32_t tile = id / ntn;
    const int32_t* tl = a.tiles + 1 + 3 * tile;
    e = tl[0], first = tl[1], rows = tl[2];
    n0 = (id - tile * ntn) * BNO;
    if constexpr (MODE == kUp) {
      if (tid < L::BM) {
        const int p = a.list[first + min(tid, rows - 1)];
        tok[tid] = p / a.k;
        wt[tid] = a.weights[p];
      }
      __syncthreads();
    }
    const int64_t ldw = (int64_t)a.K * L::WROW / L::KB, wrow = (int64_t)e * a.N + n0;
    const uint8_t* x = a.x - 2 * pad;
    if constexpr (MODE == kDown) x += first * a.ldx;
    const int64_t wo = wrow * ldw - pad * L::WROW / L::KB, so = wrow * a.lds;
    const smla_tile::Source src{x, {a.w[0].w + wo, a.w[1].w + wo}, {a.w[0].s + so, a.w[1].s + so}, (uint32_t)ldw, (uint32_t)a.lds, pad};
    uint8_t* y = a.y + first * a.ldy * (YDT == SMLA_BF16 ? 2 : 4);
    const int mine = rows - L::WM * (wave / L::NWN);
    if (mine > 32 * (L::MB - 1)) tile_body<L, MODE, YDT, L::MB>(a, lds, src, nk, rows, n0, y, tok, wt);
    else if (mine <= 0) tile_body<L, MODE, YDT, 0>(a, lds, src, nk, rows, n0, y, tok, wt);
    else if constexpr (L::MB == 2) tile_body<L, MODE, YDT, 1>(a, lds, src, nk, rows, n0, y, tok, wt);
  }
}

template <class L, int MODE, int YDT>
int launch_tile(const TileArgs& a, int64_t wgs, hipStream_t st) {
  auto kern = tile_kernel<L, MODE, YDT>;
  constexpr int lds = L::LDS + 8 * L::BM;
  static_assert(lds <= 160 * 1024, "fits a CU");
  static std::atomic<uint64_t> attr{0};
  if (hipError_t e = smla_set_dynamic_lds((const void*)kern, lds, attr); e != hipSuccess) return (int)e;
  if (wgs > 0x7fffffff) return SMLA_E_UNSUPPORTED;
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(L::THREADS), lds, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

int64_t up16(int64_t n) { return (n + 15) & ~(int64_t)15; }
int64_t padded_row(int64_t K) { return (K + 127) / 128 * 4; }  // bytes of a row of scales of whole steps

int launch_pad(const uint8_t* s, int64_t rows, int64_t K, uint8_t* out, hipStream_t st) {
  const int64_t n = rows * (padded_row(K) / 4);
  if ((n + 255) / 256 > 0x7fffffff) return SMLA_E_UNSUPPORTED;
  hipLaunchKernelGGL(pad_scales_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, s, rows, (int)(K / 32), (int)padded_row(K), out);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

// ---- y = x W^T

struct LinearPlan {
  int form, splits;  // form -1: few tokens
};

LinearPlan linear_plan(int64_t T, int64_t N, int64_t K) {
  if (T <= kFew) return {-1, 1};
  const int64_t cus = smla_num_cus(), steps = (K + 127) / 128;
  const int form = T <= 32 ? 0 : T <= 64 ? 1 : T * N >= 128 * 512 * cus ? 3 : 2;
  const int64_t tiles = (T + kFormBM[form] - 1) / kFormBM[form] * ((N + kFormBN[form] - 1) / kFormBN[form]);
  int64_t splits = 1;
  while (splits < 8 && tiles * splits * 2 <= cus && steps / (splits * 2) >= 4) splits *= 2;
  return {form, (int)splits};
}

struct LinearBytes {
  int64_t part, scales;
};
LinearBytes linear_bytes(int64_t T, int64_t N, int64_t K) {
  const LinearPlan p = linear_plan(T, N, K);
  if (p.form < 0) return {0, 0};
  return {p.splits > 1 ? up16(4 * p.splits * T * N) : 0, K % 128 ? up16(N * padded_row(K)) : 0};
}

int check_linear_fp4(int64_t T, int64_t N, int64_t K) {
  if (T < 0 || N <= 0 || K <= 0) return SMLA_E_SHAPE;
  if (K % 32 != 0 || T > (1 << 24) || N > (1 << 24) || K > (1 << 22)) return SMLA_E_UNSUPPORTED;
  return SMLA_OK;
}

template <int NW>
int launch_linear_few(const void* x, int64_t ldx, const Matrix& w, int64_t T, int64_t N, int64_t K, void* y, int y_dtype, hipStream_t st) {
  auto kern = y_dtype == SMLA_BF16 ? linear_few_kernel<NW, SMLA_BF16> : linear_few_kernel<NW, SMLA_F32>;
  hipLaunchKernelGGL(kern, dim3((unsigned)((N + 15) / 16)), dim3(64 * NW), 0, st, (const uint16_t*)x, ldx, w, (int)T, (int)N, (int)K, y);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

// ---- the experts

int check_experts(int64_t T, int64_t k, int64_t E, int64_t K, int64_t I) {
  if (T <= 0 || k <= 0 || E <= 0 || K <= 0 || I <= 0) return SMLA_E_SHAPE;
  if (K % 32 != 0 || I % 32 != 0 || E > kMaxExperts || k > kMaxChoices || K > (1 << 20) || I > (1 << 20) || T > (1 << 20) / k)
    return SMLA_E_UNSUPPORTED;
  return SMLA_OK;
}

// the tile form by the pairs an expert has on average (-1: few tokens)
int expert_form(int64_t T, int64_t k, int64_t E) {
  if (T <= kFew) return -1;
  const int64_t P = T * k, per = P / (E < P ? E : P);
  return per <= 24 ? 0 : per <= 48 ? 1 : 2;
}
int64_t max_tiles(int64_t P, int64_t E, int tile) { return P / tile + (E < P ? E : P); }

struct ExpertBytes {
  int64_t list, tiles, h, part, up_scales, down_scales;
  int64_t total() const { return 2 * list + tiles + h + part + 2 * up_scales + down_scales; }
};
ExpertBytes expert_bytes(int64_t T, int64_t k, int64_t E, int64_t K, int64_t I, bool fp4) {
  const int64_t P = T * k;
  const int form = expert_form(T, k, E);
  if (form < 0) return {0, 0, up16(2 * P * I), 0, 0, 0};
  return {up16(4 * P), up16(4 + 12 * max_tiles(P, E, kFormBM[form])), up16(2 * P * I), up16(4 * P * K),
          fp4 && K % 128 ? up16(E * I * padded_row(K)) : 0, fp4 && I % 128 ? up16(E * K * padded_row(I)) : 0};
}

template <int WT>
int launch_few(const ExpertArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(few_up_kernel<WT>, dim3(a.I / 16, a.P), dim3(64 * kUpWaves), 0, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  hipLaunchKernelGGL(few_down_kernel<WT>, dim3(a.K / 16), dim3(64 * kDownWaves), 0, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

template <class L>
int launch_tiles(const ExpertArgs& a, int64_t up_lds, int64_t down_lds, hipStream_t st) {
  const int64_t nt = max_tiles(a.P, a.E, a.tile);
  const TileArgs up{(const uint8_t*)a.x, 2 * a.ldx, {a.gate, a.up}, up_lds, a.K, a.I, 0, 0, 0, 0, (uint8_t*)a.h, a.I, 0, 1,
                    a.tiles, a.list, a.weights, a.k, a.limit};
  // (a run of workgroups a XCD: room for each XCD's share rounded up)
  int rc = launch_tile<L, kUp, SMLA_BF16>(up, nt * ((a.I + L::BN / 2 - 1) / (L::BN / 2)) + kXcds, st);
  if (rc) return rc;
  const TileArgs down{(const uint8_t*)a.h, 2 * (int64_t)a.I, {a.down, a.down}, down_lds, a.I, a.K, 0, 0, 0, 0, (uint8_t*)a.part, a.K, 0, 1,
                      a.tiles, a.list, a.weights, a.k, a.limit};
  return launch_tile<L, kDown, SMLA_F32>(down, nt * ((a.K + L::BN - 1) / L::BN) + kXcds, st);
}

template <int WT>
int launch_many(const ExpertArgs& a, int form, int64_t up_lds, int64_t down_lds, hipStream_t st) {
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(1024), 0, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  const int rc = form == 0   ? launch_tiles<Form<WT, 0>>(a, up_lds, down_lds, st)
                 : form == 1 ? launch_tiles<Form<WT, 1>>(a, up_lds, down_lds, st)
                             : launch_tiles<Form<WT, 2>>(a, up_lds, down_lds, st);
  if (rc) return rc;
  for (int64_t t0 = 0; t0 < a.T; t0 += 65535) {
    ExpertArgs c = a;
    c.at += t0 * a.k, c.y += t0 * a.K;
    const unsigned n = (unsigned)(a.T - t0 < 65535 ? a.T - t0 : 65535);
    hipLaunchKernelGGL(combine_kernel, dim3((a.K / 4 + 255) / 256, n), dim3(256), 0, st, c);
    SMLA_HIP_CHECK_LAUNCH();
  }
  return SMLA_OK;
}

}  // namespace

extern "C" size_t smla_linear_fp4_workspace(int64_t T, int64_t N, int64_t K) {
  if (T == 0 || check_linear_fp4(T, N, K) != SMLA_OK) return 0;
  const LinearBytes b = linear_bytes(T, N, K);
  return (size_t)(b.part + b.scales);
}

extern "C" int smla_linear_fp4(const void* x, int64_t ldx, const uint8_t* codes, const uint8_t* scales, int64_t T, int64_t N,
                               int64_t K, void* y, int y_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  if (y_dtype != SMLA_BF16 && y_dtype != SMLA_F32) return SMLA_E_DTYPE;
  int rc = check_linear_fp4(T, N, K);
  if (rc) return rc;
  if (T > 1 && ldx < K) return SMLA_E_SHAPE;
  if (T == 0) return SMLA_OK;
  if (!x || !codes || !scales || !y) return SMLA_E_NULL;
  if (ldx % 8 != 0 || ((uintptr_t)x & 15) || ((uintptr_t)codes & 15) || (K % 128 == 0 && ((uintptr_t)scales & 3)) || ldx > (1 << 22))
    return SMLA_E_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  const LinearPlan p = linear_plan(T, N, K);
  const Matrix w{codes, scales};
  if (p.form < 0) {
    const int64_t steps = (K + 127) / 128;
    return steps <= 16   ? launch_linear_few<4>(x, ldx, w, T, N, K, y, y_dtype, st)
           : steps <= 32 ? launch_linear_few<8>(x, ldx, w, T, N, K, y, y_dtype, st)
                         : launch_linear_few<16>(x, ldx, w, T, N, K, y, y_dtype, st);
  }
  const LinearBytes b = linear_bytes(T, N, K);
  if (!usable_workspace(workspace, workspace_bytes, (size_t)(b.part + b.scales)) && b.part + b.scales > 0) return SMLA_E_WORKSPACE;
  uint8_t* part = (uint8_t*)workspace;
  if (b.scales) {
    uint8_t* padded = part + b.part;
    if ((rc = launch_pad(scales, N, K, padded, st)) != SMLA_OK) return rc;
    scales = padded;
  }
  const int64_t nt = (T + kFormBM[p.form] - 1) / kFormBM[p.form], nn = (N + kFormBN[p.form] - 1) / kFormBN[p.form];
  const int odt = p.splits > 1 ? SMLA_F32 : y_dtype;
  TileArgs a{(const uint8_t*)x, 2 * ldx, {{codes, scales}, {nullptr, nullptr}}, padded_row(K), (int)K, (int)N, (int)T, (int)nt, (int)nn,
             p.splits, p.splits > 1 ? part : (uint8_t*)y, N, T * N, 0, nullptr, nullptr, nullptr, 1, 0.f};
  a.vec = N % (odt == SMLA_BF16 ? 8 : 4) == 0 && ((uintptr_t)a.y & 15) == 0;
  const int64_t wgs = nt * nn * p.splits;
#define SMLA_LINEAR(F) \
  (odt == SMLA_BF16 ? launch_tile<Form<kFp4, F>, kLinear, SMLA_BF16>(a, wgs, st) : launch_tile<Form<kFp4, F>, kLinear, SMLA_F32>(a, wgs, st))
  rc = p.form == 0 ? SMLA_LINEAR(0) : p.form == 1 ? SMLA_LINEAR(1) : p.form == 2 ? SMLA_LINEAR(2) : SMLA_LINEAR(3);
#undef SMLA_LINEAR
  if (rc || p.splits == 1) return rc;
  const int64_t n = T * N;
  auto red = y_dtype == SMLA_BF16 ? reduce_kernel<SMLA_BF16> : reduce_kernel<SMLA_F32>;
  hipLaunchKernelGGL(red, dim3((unsigned)((n / 4 + 256) / 256)), dim3(256), 0, st, (const float*)part, p.splits, n, y);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

extern "C" size_t smla_experts_workspace(int64_t T, int64_t k, int64_t E, int64_t K, int64_t I, int w_dtype) {
  if (check_experts(T, k, E, K, I) != SMLA_OK) return 0;
  return (size_t)expert_bytes(T, k, E, K, I, w_dtype == SMLA_FP4_E2M1).total();
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
  // (32-bit offsets: a row of x from the first one, a row of a tile's weights from its first)
  if (ldx % 8 != 0 || (((uintptr_t)x | (uintptr_t)gate | (uintptr_t)up | (uintptr_t)down | (uintptr_t)y) & 15) ||
      (fp4 && (((uintptr_t)gate_scales | (uintptr_t)up_scales | (uintptr_t)down_scales) & 3)) || ldx > (1 << 20) ||
      (T > 1 && T * ldx * 2 >= (1ll << 31)))
    return SMLA_E_UNSUPPORTED;
  const ExpertBytes b = expert_bytes(T, k, E, K, I, fp4);
  if (!usable_workspace(workspace, workspace_bytes, (size_t)b.total())) return SMLA_E_WORKSPACE;
  const int64_t P = T * k;
  ExpertArgs a{(const uint16_t*)x, ldx, ids, weights, (int)T, (int)k, (int)E, (int)K, (int)I, (int)P,
               {(const uint8_t*)gate, gate_scales}, {(const uint8_t*)up, up_scales}, {(const uint8_t*)down, down_scales}, limit,
               nullptr, nullptr, nullptr, 0, nullptr, nullptr, (uint16_t*)y};
  uint8_t* ws = (uint8_t*)workspace;
  auto take = [&](int64_t n) { uint8_t* p = ws; ws += n; return p; };
  a.list = (int32_t*)take(b.list), a.at = (int32_t*)take(b.list), a.tiles = (int32_t*)take(b.tiles);
  a.h = (uint16_t*)take(b.h), a.part = (float*)take(b.part);
  hipStream_t st = (hipStream_t)stream;
  const int form = expert_form(T, k, E);
  if (form < 0) return fp4 ? launch_few<kFp4>(a, st) : launch_few<kBf16>(a, st);
  a.tile = kFormBM[form];
  if (b.up_scales) {
    for (Matrix* m : {&a.gate, &a.up}) {
      uint8_t* s = take(b.up_scales);
      if ((rc = launch_pad(m->s, E * I, K, s, st)) != SMLA_OK) return rc;
      m->s = s;
    }
  }
  if (b.down_scales) {
    uint8_t* s = take(b.down_scales);
    if ((rc = launch_pad(a.down.s, E * K, I, s, st)) != SMLA_OK) return rc;
    a.down.s = s;
  }
  return fp4 ? launch_many<kFp4>(a, form, padded_row(K), padded_row(I), st) : launch_many<kBf16>(a, form, 0, 0, st);
}
