// Products with 4-bit weights and the experts' feed-forward networks (oracle/decode_engine.py:122-133).
//
//   linear:   y[t, n] = sum_k x[t, k] W[n, k]
//   experts:  y[t] = sum_j down_e( w_tj silu(min(g, lim)) clamp(u, -lim, lim) ),  g = gate_e x_t, u = up_e x_t,
//             e = ids[t, j]; an id outside 0 .. E-1 adds nothing.
//
// Products run on the bf16 matrix cores with fp32 sums; the weights are e2m1 codes (fp4.h) or bf16.  The hidden
// row, its router weight in it, is rounded to bf16 once: it is an operand of the second product, and half a step of
// its 8 bits is what y's own rounding costs again (the norm of y's error 0.0023-0.0024 of y's; 0.0017 with fp32 hidden
// rows, whose second product would be two or three bf16 ones).
#include "expert_tile.h"
#include "fp4.h"
#include "smla_internal.h"

#include <algorithm>

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

// The kernels for few tokens know a third type: codes of rows that are no multiple of 128 weights.  Scales of whole steps
// of 128 come through LDS, 16 bytes of a row a request (a step's four bytes of 16 rows are 16 requests, as its codes are, and
// took as long: eight tokens' up products 115 against 70 us); the others byte by byte.
constexpr int kFp4Odd = 2;

using smla_attn::lds_u32x4_t;
using smla_attn::lds_u8_t;

// 32 weights of a row, and their 8 values j = 0 .. 3.  at: the first row of 16 (the same for the wave), row: this lane's.
template <int WT>
struct Block;
template <int WT>
struct BlockFp4 {
  u32x4_t c;
  uint32_t s;
  __device__ void load(const Matrix& at, uint32_t row, uint32_t K, uint32_t kb) {
    c = *(const u32x4_t*)(at.w + (row * (K / 2) + 16 * kb));
    s = WT == kFp4Odd ? at.s[row * (K / 32) + kb] : 0;
  }
  // the scale of step s's block from LDS (scales: this lane's byte at step 0, 64 bytes a step)
  __device__ void scale(const lds_u8_t* scales, int step) {
    if constexpr (WT == kFp4) s = scales[64 * step];
  }
  __device__ void keep(bool k) { c = k ? c : u32x4_t{0, 0, 0, 0}, s = k ? s : 127; }
  // waits for the loads, and with them for every copy that was requested before: LDS is read behind it
  __device__ void arrived() { asm volatile("" : "+v"(c), "+v"(s) : : "memory"); }
  __device__ bf16x8_t frag(int j) const { return to_bf16(c[j], scale_of(s)); }
  static __device__ Matrix rows(const Matrix& m, int64_t row, int K) { return {m.w + row * (K / 2), m.s + row * (K / 32)}; }
};
template <>
struct Block<kFp4> : BlockFp4<kFp4> {};
template <>
struct Block<kFp4Odd> : BlockFp4<kFp4Odd> {};
template <>
struct Block<kBf16> {
  u32x4_t c[4];
  __device__ void load(const Matrix& at, uint32_t row, uint32_t K, uint32_t kb) {
#pragma unroll
    for (int j = 0; j < 4; j++) c[j] = *(const u32x4_t*)(at.w + (row * (2 * K) + 64 * kb + 16 * j));
  }
  __device__ void scale(const lds_u8_t*, int) {}
  __device__ void keep(bool k) {
#pragma unroll
    for (int j = 0; j < 4; j++) c[j] = k ? c[j] : u32x4_t{0, 0, 0, 0};
  }
  __device__ void arrived() { asm volatile("" : "+v"(c[0]), "+v"(c[1]), "+v"(c[2]), "+v"(c[3]) : : "memory"); }
  __device__ bf16x8_t frag(int j) const { return as_bf16x8(c[j]); }
  static __device__ Matrix rows(const Matrix& m, int64_t row, int K) { return {m.w + row * (2 * (int64_t)K), nullptr}; }
};

// ---- few tokens (up to 16): the weights are streamed once, a 16-row block of W (A of the product) against all tokens
// (B: column m of lane 16 q + m is token m).  A step is 128 k: lane group q takes the 32 of block 4 s + q on both
// sides, 16 bytes of codes a lane.  The K range is cut over the waves of a workgroup, and a wave keeps the loads of the
// next steps in flight: as a step is multiplied the one that takes its registers is requested (a batch at a time, each
// waited for whole, took half as long again).

constexpr int kFew = 16;
__device__ inline void add4(f32x4_t& a, const f32x4_t& b) {
#pragma unroll
  for (int i = 0; i < 4; i++) a[i] += b[i];
}

// Steps s0 .. s1-1 in order, U in flight: load(slot, s) in order, use(slot, s).  First what U does not divide, as one batch,
// so that no load of the rest stands under a condition: the waits are for one step then (a conditional load has the
// compiler wait for all; requesting the last step again instead costs what a step costs).  A step's reads of LDS are not
// to be gathered ahead of the step before: the registers are the loads'. 
template <int U, class L, class F>
__device__ __attribute__((always_inline)) inline void rolling(int s0, int s1, L&& load, F&& use) {
  const int rest = (s1 - s0) % U;
  if (rest) {
#pragma unroll
    for (int u = 0; u < U - 1; u++)
      if (u < rest) load(u, s0 + u);
#pragma unroll
    for (int u = 0; u < U - 1; u++)
      if (u < rest) use(u, s0 + u);
    s0 += rest;
  }
  if (s0 >= s1) return;
#pragma unroll
  for (int u = 0; u < U; u++) load(u, s0 + u);
  for (; s0 + U < s1; s0 += U)
#pragma unroll
    for (int u = 0; u < U; u += 2) {
      use(u, s0 + u);
      __builtin_amdgcn_sched_barrier(0);
      if (u + 1 < U) use(u + 1, s0 + u + 1);
      load(u, s0 + u + U);
      if (u + 1 < U) load(u + 1, s0 + u + 1 + U);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
  for (int u = 0; u < U; u++) {
    use(u, s0 + u);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// the block of step s and lane group q: clamped to the last (a step's blocks past K are dropped by `keep`)
__device__ inline int block_of(int s, int q, int nb) { return min(4 * s + q, nb - 1); }

// The steps s0 .. s1-1 of a row of K bf16 to LDS (256 bytes a step, contiguous), by this wave for itself: lane l's 16 bytes of
// every 1 KB.  Bytes past the row are not copied.
__device__ inline void copy_steps(const uint16_t* row, int K, int s0, int s1, uint32_t lds) {
  const int lane = threadIdx.x & 63, end = min(256 * s1, 2 * K);
  for (int b = 256 * s0; b < end; b += 1024)
    if (b + 16 * lane < end) smla_attn::dma16((const uint8_t*)row + b + 16 * lane, lds + b - 256 * s0);
}

// The scales of steps s0 .. s1-1 of 16 rows (last: the last that exists) to LDS, 64 bytes a step, four steps a request; room
// for whole fours.
template <int WT>
__device__ inline void copy_scales(const Matrix& at, int last, int K, int s0, int s1, uint32_t lds) {
  if constexpr (WT == kFp4) {
    const int lane = threadIdx.x & 63, row = min(lane & 15, last) * (K / 32);
    for (int s = s0; s < s1; s += 4) smla_tile::dma4_s(at.s, row + 4 * min(s + (lane >> 4), s1 - 1), lds + 64 * (s - s0));
  }
}

// the x operand j of step s from LDS (x: this lane's column at step 0, 64 bytes a lane group), 0 past K
__device__ inline bf16x8_t operand(const lds_u8_t* x, int s, int j, bool drop) {
  u32x4_t v = *(const lds_u32x4_t*)(x + 256 * s + 16 * j);
  if (drop) v = u32x4_t{0, 0, 0, 0};
  return as_bf16x8(v);
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

constexpr int kRowPad = 16;  // bytes between the rows of a wave in LDS: 16 rows' columns fall in distinct banks

// LDS of a workgroup of nw waves: n rows of K, a wave's share of all of them together, then the scales of r matrices, each a
// wave's share of whole fours of steps
__host__ __device__ inline int few_steps(int K) { return (K + 127) / 128; }
__host__ __device__ inline int few_scales(int K, int nw) { return ((few_steps(K) + nw - 1) / nw + 3) / 4 * 256; }
__host__ __device__ inline int64_t few_lds(int64_t n, int K, int nw, int r) {
  return n * (256 * (int64_t)few_steps(K) + kRowPad * nw) + nw * r * (int64_t)few_scales(K, nw);
}
// matrices whose scales go through LDS
template <int WT>
constexpr int kStaged = WT == kFp4 ? 1 : 0;

// Workgroup (i, j): outputs 16 i .. of tokens 16 j .. .  One token by 4096 x 8192 (17.8 MB): 6.3-6.8 us, 2.8 TB/s: one round
// of 256 workgroups, a launch, two dependent latencies (weights; the sums through LDS) and 2.9 us of bytes.
template <int WT, int NW, int YDT>
__global__ __launch_bounds__(64 * NW) void linear_few_kernel(const uint16_t* __restrict__ x, int64_t ldx, Matrix w, int tokens, int N,
                                                             int K, void* __restrict__ y) {
  constexpr int U = 8;
  extern __shared__ __align__(16) uint8_t lds_x[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, q = lane >> 4;
  const int nb = K / 32, steps = (nb + 3) / 4, s0 = steps * wave / NW, s1 = steps * (wave + 1) / NW, n0 = blockIdx.x * 16;
  const int t0 = blockIdx.y * kFew, T = min(tokens - t0, kFew);
  x += t0 * ldx;
  lds_u8_t *mine = (lds_u8_t*)lds_x + T * (256 * s0 + kRowPad * wave), *scales = (lds_u8_t*)lds_x + few_lds(T, K, NW, 0) + wave * few_scales(K, NW);
  const int ld = 256 * (s1 - s0) + kRowPad, row = min(m, N - 1 - n0);
  const Matrix at = Block<WT>::rows(w, n0, K);
  copy_scales<WT>(at, N - 1 - n0, K, s0, s1, (uint32_t)(uintptr_t)scales);
  for (int t = 0; t < T; t++) copy_steps(x + (int64_t)t * ldx, K, s0, s1, (uint32_t)(uintptr_t)mine + t * ld);
  const lds_u8_t* xl = mine + min(m, T - 1) * ld + 64 * q - 256 * s0;  // (columns past the last token are not stored)
  const lds_u8_t* sl = scales + 4 * m + q - 64 * s0;
  Block<WT> b[U];
  f32x4_t acc[1] = {f32x4_t{0.f, 0.f, 0.f, 0.f}};
  rolling<U>(s0, s1, [&](int u, int s) __attribute__((always_inline)) { b[u].load(at, row, K, block_of(s, q, nb)); },
             [&](int u, int s) __attribute__((always_inline)) {
               b[u].arrived();  // and the copies, which went out before
               b[u].scale(sl, s);
               const bool drop = 4 * s + 4 > nb && 4 * s + q >= nb;
               if (4 * s + 4 > nb) b[u].keep(!drop);  // uniform
#pragma unroll
               for (int j = 0; j < 4; j++)
                 acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[u].frag(j), operand(xl, s, j, drop), acc[0], 0, 0, 0);
             });
  join<NW>(acc);
  if (wave != 0 || m >= T) return;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int n = n0 + 4 * q + i;
    if (n < N) {
      if constexpr (YDT == SMLA_BF16) ((uint16_t*)y)[(int64_t)(t0 + m) * N + n] = bf16_rne(acc[0][i]);
      else ((float*)y)[(int64_t)(t0 + m) * N + n] = acc[0][i];
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
  uint32_t* items;       // few tokens: [P][4], few_down_kernel's
  int32_t* list;         // pairs by expert
  int32_t* at;           // a pair's place in it
  int32_t* tiles;        // [8] their numbers, then for each XCD `room` of (expert, first place, pairs)
  int tile, room;        // pairs of a tile at most
  uint16_t* h;           // [P, I] hidden rows, by place (few tokens: by pair)
  float* part;           // [P, K] their products, by place
  uint16_t* y;
};

constexpr int kMaxExperts = 1024, kMaxChoices = 64;
constexpr int kItemTokens = 4;

// (comparisons, not fminf: a NaN stays one)
__device__ inline float gated(float g, float u, float lim) {
  g = g > lim ? lim : g, u = u > lim ? lim : u < -lim ? -lim : u;
  return g / (1.f + __expf(-g)) * u;
}

// Workgroup (i, p): 16 hidden rows' gate and up products of the expert of pair p, where p is its first pair, for the
// tokens that have it: column m is the m-th of them.  A token that has it twice has the sum of its weights.  A wave has its
// K range of the tokens' rows of x in LDS (in registers they would take three times the weights' and leave one workgroup a
// CU), room for `cap` of them; an expert of more streams its weights again for the others.
// Bound by HBM: 8 tokens x 6 of 256 experts of 4096 x 2048 (390 MB) 71-75 us, 5.3 TB/s, where a bare read of such rows reaches
// 6.2; one token 13 us.  Four, six or eight steps in flight and 2, 4 or 8 waves take the same; two blocks of 16 rows a
// workgroup, one behind the other, 2 us longer.
constexpr int kUpWaves = 4;
template <int WT>
constexpr int kUpAhead = WT == kBf16 ? 2 : 4;
template <int WT>
__global__ __launch_bounds__(64 * kUpWaves) __attribute__((amdgpu_waves_per_eu(4))) void few_up_kernel(const ExpertArgs a, int cap) {
  constexpr int U = kUpAhead<WT>;
  extern __shared__ __align__(16) uint8_t lds_x[];
  const int p = blockIdx.y, e = __builtin_amdgcn_readfirstlane(a.ids[p]), lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, q = lane >> 4;
  // lane t < T: token t's first place with this expert, and its weight; eight loads at a time (one after the other they
  // took longer than the weights)
  int pair = -1;
  float wt = 0.f;
  for (int j0 = 0; j0 < a.k; j0 += 8) {
    int id[8];
    float w[8];
    const int base = min(lane, a.T - 1) * a.k;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      id[j] = a.ids[base + min(j0 + j, a.k - 1)];
      w[j] = a.weights[base + min(j0 + j, a.k - 1)];
    }
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (lane < a.T && j0 + j < a.k && id[j] == e) {
        if (pair < 0) pair = base + j0 + j;
        wt += w[j];
      }
  }
  uint32_t has = __builtin_amdgcn_readfirstlane((uint32_t)__ballot(pair >= 0));
  const bool real = e >= 0 && e < a.E;
  if (blockIdx.x == 0 && wave == 0) {
    // few_down_kernel's item of place p: {expert | tokens << 10, their places by 16 bits}, where p is the first place of each
    // fourth token with the expert; 0: none
    const int t = p / a.k;
    uint32_t what = 0, places[2] = {0, 0};
    if (real && __builtin_amdgcn_readlane(pair, t) == p && __popc(has & ((1u << t) - 1)) % kItemTokens == 0) {
      uint32_t left = has >> t << t;
#pragma unroll
      for (int c = 0; c < kItemTokens; c++)
        if (left) {
          const int b = __ffs((int)left) - 1;
          left &= left - 1;
          what |= 1u << b;
          places[c / 2] |= (uint32_t)__builtin_amdgcn_readlane(pair, b) << (16 * (c & 1));
        }
      what = (uint32_t)e | what << 10;
    }
    if (lane == 0) *(u32x4_t*)(a.items + 4 * p) = u32x4_t{what, places[0], places[1], 0};
  }
  if (!real || __any(pair >= 0 && pair < p)) return;
  const int i0 = blockIdx.x * 16, nb = a.K / 32, steps = (nb + 3) / 4;
  const int s0 = steps * wave / kUpWaves, s1 = steps * (wave + 1) / kUpWaves, ld = 256 * (s1 - s0) + kRowPad;
  const int s_up = few_scales(a.K, kUpWaves);
  lds_u8_t *mine = (lds_u8_t*)lds_x + cap * (256 * s0 + kRowPad * wave),
           *scales = (lds_u8_t*)lds_x + few_lds(cap, a.K, kUpWaves, 0) + wave * 2 * s_up;
  const Matrix gate = Block<WT>::rows(a.gate, (int64_t)e * a.I + i0, a.K), up = Block<WT>::rows(a.up, (int64_t)e * a.I + i0, a.K);
  copy_scales<WT>(gate, 15, a.K, s0, s1, (uint32_t)(uintptr_t)scales);
  copy_scales<WT>(up, 15, a.K, s0, s1, (uint32_t)(uintptr_t)scales + s_up);
  const lds_u8_t* sl = scales + 4 * m + q - 64 * s0;
  while (has) {
    int col = 0, nt = 0;  // lane m < nt: its token
    for (; has && nt < cap; nt++) {
      const int t = __ffs((int)has) - 1;
      has &= has - 1;
      if (m == nt) col = t;
      copy_steps(a.x + t * a.ldx, a.K, s0, s1, (uint32_t)(uintptr_t)mine + nt * ld);
    }
    const lds_u8_t* xl = mine + min(m, nt - 1) * ld + 64 * q - 256 * s0;
    uint32_t wr = m, wq = q;  // (not known to be the same in every pass: else the addresses of all loads are kept, and spilled)
    asm volatile("" : "+v"(wr), "+v"(wq));
    Block<WT> w[U][2];
    f32x4_t acc[2];
    acc[0] = acc[1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    rolling<U>(s0, s1, [&](int u, int s) __attribute__((always_inline)) {
      const int kb = block_of(s, wq, nb);
      w[u][0].load(gate, wr, a.K, kb);
      w[u][1].load(up, wr, a.K, kb);
    }, [&](int u, int s) __attribute__((always_inline)) {
      w[u][0].arrived();  // and the copies, which went out before
      w[u][1].arrived();
      w[u][0].scale(sl, s);
      w[u][1].scale(sl + s_up, s);
      const bool drop = 4 * s + 4 > nb && 4 * s + q >= nb;
      if (4 * s + 4 > nb) {  // uniform
        w[u][0].keep(!drop);
        w[u][1].keep(!drop);
      }
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const bf16x8_t x = operand(xl, s, j, drop);
#pragma unroll
        for (int r = 0; r < 2; r++) acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[u][r].frag(j), x, acc[r], 0, 0, 0);
      }
    });
    join<kUpWaves>(acc);
    const int to = __shfl(pair, col, 64);
    const float weight = __shfl(wt, col, 64);
    if (wave == 0 && m < nt) {
      float h[4];
#pragma unroll
      for (int i = 0; i < 4; i++) h[i] = weight * gated(acc[0][i], acc[1][i], a.limit);
      *(u32x2_t*)(a.h + (int64_t)to * a.I + i0 + 4 * q) = u32x2_t{pack_bf16x2(h[0], h[1]), pack_bf16x2(h[2], h[3])};
    }
    if (has) __syncthreads();  // the sums are read before the next pass writes its own
  }
}

// Workgroup i: 16 columns of y for every token, over all experts that any token has: the waves share out the K
// ranges of all of them.  An item is an expert and up to kItemTokens tokens that have it, whose hidden rows go to the
// wave's LDS a step ahead of the step's weights (256 bytes a token; as operands from memory they are four loads of 1 KB
// a step, against one of the weights).  Column m is token m: a wave adds an item's sums to a token's only where the item
// has it (0 times an infinite weight of another token's expert would be NaN).
// The items come from few_up_kernel, which has the tokens of each expert at hand: listing them here took 2 us of every
// workgroup.  8 tokens x 6 experts (200 MB) 41-45 us, 4.7 TB/s (with each step requested alone, half a 128-byte line a row,
// 45-46; three to five steps in flight are alike); one token 8.7 us.
constexpr int kDownWaves = 16;
template <int WT>
constexpr int kDownAhead = WT == kBf16 ? 3 : 4;
template <int WT>
constexpr int kDownRing = kDownAhead<WT> * kItemTokens * 256;
template <int WT>
constexpr int kDownScales = WT == kFp4 ? (kDownAhead<WT> + 2) * 256 : 0;
template <int WT>
constexpr int kDownLds = kDownWaves * (kDownRing<WT> + kDownScales<WT>);

template <int WT>
__global__ __launch_bounds__(64 * kDownWaves) void few_down_kernel(const ExpertArgs a) {
  constexpr int U = kDownAhead<WT>;
  extern __shared__ __align__(16) uint8_t lds_x[];
  __shared__ u32x4_t item[kFew * kMaxChoices];
  __shared__ int cnt[kDownWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, q = lane >> 4;
  // the items, in the order of their places
  u32x4_t mine = {0, 0, 0, 0};
  if (tid < a.P) mine = *(const u32x4_t*)(a.items + 4 * tid);
  const uint64_t mask = __ballot(mine[0] != 0);
  if (lane == 0) cnt[wave] = __popcll(mask);
  __syncthreads();
  int to = __popcll(mask & ((1ull << lane) - 1)), items = 0;
  for (int v = 0; v < kDownWaves; v++) {
    if (v < wave) to += cnt[v];
    items += cnt[v];
  }
  if (mine[0]) item[to] = mine;
  __syncthreads();
  items = __builtin_amdgcn_readfirstlane(items);

  const int n0 = blockIdx.x * 16, nb = a.I / 32, per = (nb + 3) / 4, steps = items * per;
  const int s0 = steps * wave / kDownWaves & ~1, s1 = wave + 1 == kDownWaves ? steps : steps * (wave + 1) / kDownWaves & ~1;
  lds_u8_t *ring = (lds_u8_t*)lds_x + wave * kDownRing<WT>, *scales = (lds_u8_t*)lds_x + kDownWaves * kDownRing<WT> + wave * kDownScales<WT>;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f}, acc = sum;
  int lk = s0 % per, uk = lk, li = s0 / per, ui = li;  // an item's step, and the item, of the loads and of the products
  auto get = [&](int i) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(i < items ? item[i][0] : 0); };
  uint32_t lit = get(li), uit = lit;
  auto places = [&](int i, int c) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(i < items ? item[i][1 + c] : 0); };
  // scales: a request for each four steps of an item that the wave has any of, in a ring of slots of 256 bytes
  constexpr int SLOTS = U + 2;
  int ls = -1, us = -1;  // slots of the loads' and the products' step
  auto next = [&](int slot) __attribute__((always_inline)) { return slot + 1 == SLOTS ? 0 : slot + 1; };
  uint32_t lp0 = places(li, 0), lp1 = places(li, 1);  // the places of the loads' item
  Block<WT> w[U];
  rolling<U>(s0, s1, [&](int u, int s) __attribute__((always_inline)) {
    const uint32_t ex = lit & 1023;
    const Matrix at = Block<WT>::rows(a.down, (int64_t)ex * a.K + n0, a.I);
    const int many = __popc(lit >> 10);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot's last reads are done
    for (int c = 0; c < many; c++) {  // uniform
      const uint32_t pair = (c < 2 ? lp0 : lp1) >> (16 * (c & 1)) & 0xffff;
      const int b = min(256 * lk + 4 * lane, 2 * a.I - 4);  // (past the row: any, dropped)
      smla_tile::dma4_s((const uint8_t*)a.h + 2 * (int64_t)pair * a.I, b, (uint32_t)(uintptr_t)ring + (u * kItemTokens + c) * 256);
    }
    if constexpr (WT == kFp4) {
      if (lk % 4 == 0 || s == s0) {  // uniform
        ls = next(ls);
        smla_tile::dma4_s(at.s, m * (a.I / 32) + 4 * min((lk & ~3) + q, per - 1), (uint32_t)(uintptr_t)scales + 256 * ls);
      }
    }
    w[u].load(at, m, a.I, block_of(lk, q, nb));
    if (++lk == per) lk = 0, lit = get(++li), lp0 = places(li, 0), lp1 = places(li, 1);
  }, [&](int u, int s) __attribute__((always_inline)) {
    w[u].arrived();  // and the copies, which went out before
    if (uk % 4 == 0 || s == s0) us = next(us);
    w[u].scale(scales + 256 * us + 4 * m + q, uk & 3);
    const bool drop = 4 * uk + 4 > nb && 4 * uk + q >= nb;
    if (4 * uk + 4 > nb) w[u].keep(!drop);  // uniform
    const uint32_t has = uit >> 10;
    const lds_u8_t* x = ring + (u * kItemTokens + min((int)__popc(has & ((1u << m) - 1)), kItemTokens - 1)) * 256 + 64 * q;
#pragma unroll
    for (int j = 0; j < 4; j++) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[u].frag(j), operand(x, 0, j, drop), acc, 0, 0, 0);
    if (++uk == per || s + 1 == s1) {
      if (has >> m & 1) add4(sum, acc);
      acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
      uk = 0, uit = get(++ui);
    }
  });
  f32x4_t all[1] = {sum};
  __syncthreads();
  join<kDownWaves>(all);
  if (wave != 0 || m >= a.T) return;
  *(u32x2_t*)(a.y + (int64_t)m * a.K + n0 + 4 * q) = u32x2_t{pack_bf16x2(all[0][0], all[0][1]), pack_bf16x2(all[0][2], all[0][3])};
}

// ---- more tokens: the pairs (token, choice) sorted by expert, in tiles of one expert's pairs.

template <class F>
__device__ inline void each_pair(const ExpertArgs& a, F&& f) {
  constexpr int U = 12;  // ids in flight a thread (one after the other: 33 us for 4096 tokens of 6, against 24)
  for (int p0 = threadIdx.x; p0 < a.P; p0 += 1024 * U) {
    int e[U];
#pragma unroll
    for (int u = 0; u < U; u++) e[u] = a.ids[min(p0 + 1024 * u, a.P - 1)];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (p0 + 1024 * u < a.P) f(p0 + 1024 * u, e[u]);
  }
}

// An expert's pairs go to tiles by twos, which share its weights in an XCD's L2.  Such units go to the XCDs in turn, the
// longest first: every XCD has as many of each length (tiles in the experts' order, an eighth of them an XCD, left one with
// up to a sixth more to do than the others; the short ones last fill the end).  The order within an expert and among units of
// a length is as it comes; no result depends on it.
constexpr int kMaxPairs = 1 << 20;
constexpr int kMaxUnits = kMaxPairs / 256 + kMaxExperts;  // (tiles of 32 pairs are taken for 32 an expert and less)
__global__ __launch_bounds__(1024) void plan_kernel(const ExpertArgs a) {
  __shared__ int cnt[kMaxExperts], part[16], length[16], units_of[16];
  __shared__ int unit_at[kMaxUnits], unit[kMaxUnits];  // first place; expert | pairs << 10
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  cnt[tid] = 0;
  if (tid < 16) length[tid] = units_of[tid] = 0;
  __syncthreads();
  each_pair(a, [&](int, int e) {
    if (e >= 0 && e < a.E) atomicAdd(&cnt[e], 1);
  });
  __syncthreads();
  const int n = cnt[tid], upto = wave_incl_scan(n);
  if (lane == 63) part[wave] = upto;
  // units by their length in 32s (1 .. most)
  const int most = 2 * a.tile / 32, whole = n / (2 * a.tile), rest = n - whole * 2 * a.tile, of_rest = (rest + 31) / 32;
  if (whole) atomicAdd(&length[most], whole);
  if (rest) atomicAdd(&length[of_rest], 1);
  __syncthreads();
  int first = upto - n;
  for (int v = 0; v < wave; v++) first += part[v];
  auto place = [&](int len, int many) {
    int at = atomicAdd(&units_of[len], many);
    for (int l = len + 1; l <= most; l++) at += length[l];
    return at;
  };
  if (whole) {
    const int at = place(most, whole);
    for (int i = 0; i < whole; i++) unit_at[at + i] = first + 2 * a.tile * i, unit[at + i] = tid | (2 * a.tile) << 10;
  }
  if (rest) {
    const int at = place(of_rest, 1);
    unit_at[at] = first + n - rest, unit[at] = tid | rest << 10;
  }
  cnt[tid] = first;
  __syncthreads();
  if (wave < kXcds) {  // an XCD's tiles
    int units = 0, base = 0;
    for (int l = 1; l <= most; l++) units += length[l];
    for (int u0 = 0; kXcds * u0 < units; u0 += 64) {
      const int u = kXcds * (u0 + lane) + wave;
      const int what = u < units ? unit[u] : 0, pairs = what >> 10, tiles = (pairs + a.tile - 1) / a.tile;
      const int to = base + wave_incl_scan(tiles) - tiles;
      for (int i = 0; i < tiles; i++) {
        int32_t* t = a.tiles + 8 + 3 * ((int64_t)wave * a.room + to + i);
        t[0] = what & 1023, t[1] = unit_at[u] + i * a.tile, t[2] = min(a.tile, pairs - i * a.tile);
      }
      base = __shfl(to + tiles, 63, 64);
    }
    if (lane == 0) a.tiles[wave] = base;
  }
  each_pair(a, [&](int p, int e) {
    const bool real = e >= 0 && e < a.E;
    const int i = real ? atomicAdd(&cnt[e], 1) : -1;
    if (real) a.list[i] = p;
    a.at[p] = i;
  });
}

// y[t] = the sum of its pairs' rows, in their order.  Bound by HBM: 24576 rows of 4096 (403 MB) 80 us, 5.4 TB/s with y.  The rows
// are fp32: bf16 ones would halve that, and round each of a token's k products as coarsely as y.
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

// tokens x outputs, waves of .. x .., stages, k of a step.  Few tokens an expert stream the weights: 128 bytes of a row
// a copy (64 bytes a step, with every row in turn, come at 4.9 TB/s, 128 at 6.2).  64 x 128 is for the sizes between, whose
// large tiles are too few for the CUs.
template <int WT, int FORM>
struct Form;
template <>
struct Form<kFp4, 0> : smla_tile::Tile<kFp4, 32, 256, 32, 64, 3, 256> {};  // 156 KB, 4 waves
template <>
struct Form<kFp4, 1> : smla_tile::Tile<kFp4, 64, 128, 32, 64, 3, 128> {};  // 78 KB, 4 waves: two workgroups a CU
template <>
struct Form<kFp4, 2> : smla_tile::Tile<kFp4, 128, 512, 64, 128, 2, 128> {};  // 152 KB, 8 waves
template <>
struct Form<kBf16, 1> : smla_tile::Tile<kBf16, 64, 128, 32, 64, 3, 64> {};  // 72 KB, 4 waves: two workgroups a CU
template <>
struct Form<kBf16, 2> : smla_tile::Tile<kBf16, 128, 256, 64, 64, 3, 64> {};  // 144 KB, 8 waves
constexpr int kForms = 3;
constexpr int kFormBM[kForms] = {32, 64, 128}, kFormBN[kForms] = {256, 128, 512}, kFormKB[kForms] = {256, 128, 128};  // (BN, KB: kFp4)

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
  int room;
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

// Figures.  4-bit, 128 x 512: 4096 x 4096 x 8192 in 186-196 us, 1.40-1.48 PFLOP/s (an 8192^3 bf16 library product: 1.29), bound by
// the products; 256 experts of 4096 x 2048 with 96 pairs each, the up products 805 us, 1.02 PFLOP/s (128 each 1.17, 256 each 1.3:
// what a tile lacks of its rows costs about as much as what is there).  32 x 256: 100 tokens x 6 of those experts, up 371-460
// and down 195-239 us for 3.1 GB, bound by HBM at 5.2-5.4 TB/s over the call.  bf16: 24 experts of 2048 x 1408, 1000 pairs, up
// 84 us and down 32 for 415 MB: 264 tiles leave 8 CUs with two.
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
                                {a.w[0].s + (int64_t)n0 * a.lds + (s0 ? 4 * (s0 * (L::KB / 128) - pad / 128) : 0), nullptr},
                                (uint32_t)(a.K * L::WROW / L::KB), (uint32_t)a.lds, s0 == 0 ? pad : 0};
    uint8_t* y = a.y + (sp * a.split_stride + first * a.ldy) * (YDT == SMLA_BF16 ? 2 : 4);
    const int mine = rows - L::WM * (wave / L::NWN);
    if (mine > 32 * (L::MB - 1)) tile_body<L, MODE, YDT, L::MB>(a, lds, src, nk, rows, n0, y, tok, wt);
    else if (mine <= 0) tile_body<L, MODE, YDT, 0>(a, lds, src, nk, rows, n0, y, tok, wt);
    else if constexpr (L::MB == 2) tile_body<L, MODE, YDT, 1>(a, lds, src, nk, rows, n0, y, tok, wt);
  } else {
    // workgroups are dealt to the XCDs in turn: this XCD's tiles, all of a tile's columns one after the other
    const uint32_t ntn = (a.N + BNO - 1) / BNO, xcd = blockIdx.x % kXcds, id = blockIdx.x / kXcds, tile = id / ntn;
    if (tile >= (uint32_t)a.tiles[xcd]) return;
    const int32_t* tl = a.tiles + 8 + 3 * (xcd * a.room + tile);
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
  if (wgs * L::THREADS > 0xffffffff) return SMLA_E_UNSUPPORTED;
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(L::THREADS), lds, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

int64_t up16(int64_t n) { return (n + 15) & ~(int64_t)15; }
int64_t padded_row(int64_t K) { return (K + 127) / 128 * 4; }  // bytes of a row of scales of whole steps

int launch_pad(const uint8_t* s, int64_t rows, int64_t K, uint8_t* out, hipStream_t st) {
  const int64_t n = rows * (padded_row(K) / 4);
  if (n > 0xffffff00) return SMLA_E_UNSUPPORTED;
  hipLaunchKernelGGL(pad_scales_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, s, rows, (int)(K / 32), (int)padded_row(K), out);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

// ---- y = x W^T

constexpr int kMaxFewLds = 144 * 1024;  // the tokens' rows (and up to 16 KB of sums)

struct LinearPlan {
  int form, splits;  // form -1: few tokens
};

// waves of the kernel for few tokens: about four steps of 128 k each
int few_waves(int64_t K) { return K <= 2048 ? 4 : K <= 4096 ? 8 : 16; }

LinearPlan linear_plan(int64_t T, int64_t N, int64_t K) {
  // A model of the launches in microseconds, its constants fitted to 112 products (T 17 .. 512, N 256 .. 16384, K 512 .. 4096):
  // the plan it picks is 2 % off the fastest on average and 30 % at worst among those; larger sizes go by the same model,
  // extrapolated.  The kernel for few tokens: a workgroup's time
  // goes with the bytes it reads (16 tokens and 16 outputs), those resident together overlap.  Tiles: a step takes kIdle when
  // few CUs run, kOne with a workgroup on each, kBusy with as many as fit; a split adds the launch that sums and its
  // fp32 partial sums, rows of scales that are no whole words another that lays them out.
  constexpr double kIdle[kForms] = {0.95, 0.46, 2.2}, kOne[kForms] = {1.25, 0.66, 2.85}, kBusy[kForms] = {1.25, 1.08, 2.85};
  const int64_t cus = smla_num_cus();
  LinearPlan best{kForms - 1, 1};
  double bt = 1e30;
  const int nw = few_waves(K);
  const int64_t cols = std::min<int64_t>(T, kFew), lds = few_lds(cols, (int)K, nw, K % 128 == 0);
  const int64_t tt = (T + kFew - 1) / kFew;
  if (lds <= kMaxFewLds && tt <= 65535) {  // (the grid's limit)
    const int64_t wgs = (N + 15) / 16 * tt;
    const double each = std::max(0.7, K * (2.0 * T / tt + 8.5) * 25.3e-6);
    const bool alone = 2 * (lds + 1024 * nw) > 160 * 1024;  // on a CU
    const double more = alone ? (double)((wgs + cus - 1) / cus - 1) : std::max(0.0, (double)wgs / cus - 1);
    bt = 3.6 + 0.35 * K / 1024 + more * each;
    best = {-1, 1};
  }
  for (int f = 0; f < kForms; f++) {
    const int64_t tiles = (T + kFormBM[f] - 1) / kFormBM[f] * ((N + kFormBN[f] - 1) / kFormBN[f]), steps = (K + kFormKB[f] - 1) / kFormKB[f];
    const int64_t cap = f == 1 ? 2 * cus : cus;
    for (int s = 1; s <= (f == 2 ? 1 : 8) && (s == 1 || steps / s >= 2); s *= 2) {  // (large tiles are for many)
      const int64_t rest = tiles * s % cap;
      double t = (double)(tiles * s / cap) * kBusy[f];
      if (rest > cus) t += kOne[f] + (kBusy[f] - kOne[f]) * (double)(rest - cus) / (double)cus;
      else if (rest > 0) t += kIdle[f] + (kOne[f] - kIdle[f]) * (double)rest / (double)cus;
      t = 3.6 + t * (double)((steps + s - 1) / s);
      t = std::max(t, 2.5 + N * (double)K * 0.53 / 5.5e6);
      if (s > 1) t += 2.4 + s * (double)T * N * 8 / 4.3e6;
      if (K % 128) t += 2.5;
      if (t < bt) bt = t, best = {f, s};
    }
  }
  return best;
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

template <int WT, int NW>
int launch_linear_few(const void* x, int64_t ldx, const Matrix& w, int64_t T, int64_t N, int64_t K, void* y, int y_dtype, hipStream_t st) {
  const bool bf = y_dtype == SMLA_BF16;
  auto kern = bf ? linear_few_kernel<WT, NW, SMLA_BF16> : linear_few_kernel<WT, NW, SMLA_F32>;
  static std::atomic<uint64_t> attr[2] = {{0}, {0}};
  if (hipError_t e = smla_set_dynamic_lds((const void*)kern, kMaxFewLds, attr[bf]); e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(kern, dim3((unsigned)((N + 15) / 16), (unsigned)((T + kFew - 1) / kFew)), dim3(64 * NW),
                     few_lds(std::min<int64_t>(T, kFew), (int)K, NW, kStaged<WT>), st, (const uint16_t*)x, ldx, w,
                     (int)T, (int)N, (int)K, y);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

// ---- the experts

int check_experts(int64_t T, int64_t k, int64_t E, int64_t K, int64_t I) {
  if (T <= 0 || k <= 0 || E <= 0 || K <= 0 || I <= 0) return SMLA_E_SHAPE;
  if (K % 32 != 0 || I % 32 != 0 || E > kMaxExperts || k > kMaxChoices || K > (1 << 20) || I > (1 << 20) || T > kMaxPairs / k)
    return SMLA_E_UNSUPPORTED;
  return SMLA_OK;
}

// The tile form by the pairs an expert has on average (-1: few tokens).  4-bit weights in 64 x 128 tiles came out behind
// one of the others at every number of pairs (256 experts of 4096 x 2048, the up products: 48 pairs 709 us, 128 x 512 696;
// 32 pairs 640, 32 x 256 513).  bf16 in 32 x 256 tiles came out behind 64 x 128 at every number (24 experts of 4096 x 2048:
// 8 pairs 247 us against 235, 48 pairs 271 against 247); 128 x 256 passes those between 48 (261) and 64 (256 against 278).
// The average is of all T k pairs over the E experts here, which the host knows without the ids: it is too high by the share of
// ids outside 0 .. E-1 (24 of 48 experts here: 83 for 42, 128 x 256 in 126-131 us where 64 x 128 takes 117), and a shared expert's
// pairs, T of them, count as any other's (1000 tokens of 256 + 1 experts: 32 x 256 throughout).  K, I and the number of CUs play no
// part: 8 experts of 4096 x 1024 with 128 pairs each are 32 and 64 workgroups (79 and 27 us).
// Few tokens: the LDS test is for T rows, though few_up_kernel holds `cap` of them.
int expert_form(int64_t T, int64_t k, int64_t E, int64_t K, bool fp4) {
  if (T <= kFew && few_lds(T, (int)K, kUpWaves, 2) <= kMaxFewLds) return -1;
  const int64_t P = T * k, per = P / (E < P ? E : P);
  return fp4 ? per <= 32 ? 0 : 2 : per <= 56 ? 1 : 2;
}
// an XCD's tiles at most: units of one length are shared out evenly (plan_kernel)
int64_t room_of(int64_t P, int64_t E, int tile) { return (P / tile + (E < P ? E : P)) / kXcds + 3; }

struct ExpertBytes {
  int64_t items, list, tiles, h, part, up_scales, down_scales;
  int64_t total() const { return items + 2 * list + tiles + h + part + 2 * up_scales + down_scales; }
};
ExpertBytes expert_bytes(int64_t T, int64_t k, int64_t E, int64_t K, int64_t I, bool fp4) {
  const int64_t P = T * k;
  const int form = expert_form(T, k, E, K, fp4);
  if (form < 0) return {16 * P, 0, 0, up16(2 * P * I), 0, 0, 0};
  return {0, up16(4 * P), up16(32 + 12 * kXcds * room_of(P, E, kFormBM[form])), up16(2 * P * I), up16(4 * P * K),
          fp4 && K % 128 ? up16(E * I * padded_row(K)) : 0, fp4 && I % 128 ? up16(E * K * padded_row(I)) : 0};
}

template <int WT>
int launch_few_up(const ExpertArgs& a, hipStream_t st) {
  // rows for four times the tokens that an expert has on average, and two more; one that all tokens have (a shared one) is
  // streamed once for each `cap` of them: 256 experts of 4096 x 2048 and a shared one, 6 + 1 a token, up and down: 8 tokens (cap 2) 94
  // and 55 us, 16 (cap 3) 155 and 88
  const int cap = (int)std::min<int64_t>(a.T, 4 * a.P / a.E + 2), lds = (int)few_lds(cap, a.K, kUpWaves, 2 * kStaged<WT>);
  static std::atomic<uint64_t> attr{0};
  if (hipError_t e = smla_set_dynamic_lds((const void*)few_up_kernel<WT>, kMaxFewLds, attr); e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(few_up_kernel<WT>, dim3(a.I / 16, a.P), dim3(64 * kUpWaves), lds, st, a, cap);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

template <int WT>
int launch_few_down(const ExpertArgs& a, hipStream_t st) {
  static std::atomic<uint64_t> attr2{0};
  if (hipError_t e = smla_set_dynamic_lds((const void*)few_down_kernel<WT>, kDownLds<WT>, attr2); e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(few_down_kernel<WT>, dim3(a.K / 16), dim3(64 * kDownWaves), kDownLds<WT>, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

int launch_few(const ExpertArgs& a, bool fp4, hipStream_t st) {
  int rc = !fp4 ? launch_few_up<kBf16>(a, st) : a.K % 128 ? launch_few_up<kFp4Odd>(a, st) : launch_few_up<kFp4>(a, st);
  if (rc) return rc;
  return !fp4 ? launch_few_down<kBf16>(a, st) : a.I % 128 ? launch_few_down<kFp4Odd>(a, st) : launch_few_down<kFp4>(a, st);
}

template <class L>
int launch_tiles(const ExpertArgs& a, int64_t up_lds, int64_t down_lds, hipStream_t st) {
  const int64_t nt = kXcds * (int64_t)a.room;
  const TileArgs up{(const uint8_t*)a.x, 2 * a.ldx, {a.gate, a.up}, up_lds, a.K, a.I, 0, 0, 0, 0, (uint8_t*)a.h, a.I, 0, 1,
                    a.tiles, a.room, a.list, a.weights, a.k, a.limit};
  const int rc = launch_tile<L, kUp, SMLA_BF16>(up, nt * ((a.I + L::BN / 2 - 1) / (L::BN / 2)), st);
  if (rc) return rc;
  const TileArgs down{(const uint8_t*)a.h, 2 * (int64_t)a.I, {a.down, a.down}, down_lds, a.I, a.K, 0, 0, 0, 0, (uint8_t*)a.part, a.K, 0, 1,
                      a.tiles, a.room, a.list, a.weights, a.k, a.limit};
  return launch_tile<L, kDown, SMLA_F32>(down, nt * ((a.K + L::BN - 1) / L::BN), st);
}

template <int WT>
int launch_many(const ExpertArgs& a, int form, int64_t up_lds, int64_t down_lds, hipStream_t st) {
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(1024), 0, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  int rc = SMLA_OK;
  if (form < 2) rc = launch_tiles<Form<WT, WT == kFp4 ? 0 : 1>>(a, up_lds, down_lds, st);
  else rc = launch_tiles<Form<WT, 2>>(a, up_lds, down_lds, st);
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
  if (ldx % 8 != 0 || (((uintptr_t)x | (uintptr_t)codes | (uintptr_t)y) & 15) || (K % 128 == 0 && ((uintptr_t)scales & 3)) || ldx > (1 << 22))
    return SMLA_E_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  const LinearPlan p = linear_plan(T, N, K);
  const Matrix w{codes, scales};
  if (p.form < 0) {
    const int nw = few_waves(K);
#define SMLA_FEW(WT)                                                              \
  (nw == 4   ? launch_linear_few<WT, 4>(x, ldx, w, T, N, K, y, y_dtype, st)     \
   : nw == 8 ? launch_linear_few<WT, 8>(x, ldx, w, T, N, K, y, y_dtype, st)     \
             : launch_linear_few<WT, 16>(x, ldx, w, T, N, K, y, y_dtype, st))
    return K % 128 ? SMLA_FEW(kFp4Odd) : SMLA_FEW(kFp4);
#undef SMLA_FEW
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
             p.splits, p.splits > 1 ? part : (uint8_t*)y, N, T * N, 0, nullptr, 0, nullptr, nullptr, 1, 0.f};
  a.vec = N % (odt == SMLA_BF16 ? 8 : 4) == 0;
  const int64_t wgs = nt * nn * p.splits;
#define SMLA_LINEAR(F) \
  (odt == SMLA_BF16 ? launch_tile<Form<kFp4, F>, kLinear, SMLA_BF16>(a, wgs, st) : launch_tile<Form<kFp4, F>, kLinear, SMLA_F32>(a, wgs, st))
  rc = p.form == 0 ? SMLA_LINEAR(0) : p.form == 1 ? SMLA_LINEAR(1) : SMLA_LINEAR(2);
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
               nullptr, nullptr, nullptr, nullptr, 0, 0, nullptr, nullptr, (uint16_t*)y};
  uint8_t* ws = (uint8_t*)workspace;
  auto take = [&](int64_t n) { uint8_t* p = ws; ws += n; return p; };
  a.items = (uint32_t*)take(b.items), a.list = (int32_t*)take(b.list), a.at = (int32_t*)take(b.list), a.tiles = (int32_t*)take(b.tiles);
  a.h = (uint16_t*)take(b.h), a.part = (float*)take(b.part);
  hipStream_t st = (hipStream_t)stream;
  const int form = expert_form(T, k, E, K, fp4);
  if (form < 0) return launch_few(a, fp4, st);
  a.tile = kFormBM[form], a.room = (int)room_of(P, E, a.tile);
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
