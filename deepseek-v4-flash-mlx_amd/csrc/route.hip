// Routing of tokens to experts (oracle/decode_engine.py:122-128: scores, the balance bias, the top-k, its
// weights).
//
//   s_e = softmax | sigmoid | sqrt(softplus) of the logits;  r_e = s_e + bias_e
//   a group of E / groups experts is worth the sum of its two largest r; the topk_groups best stay
//   ids = the k largest r that stay, in that order; w_j = s[ids_j] (/ their sum) * scale
//
// Ties go to the lowest id, and the order is that of the values and not of their fp32 roundings: two scores an
// fp32 step apart would otherwise trade places with the formula's rounding.  Without a bias the scores' order
// is the logits', which needs no scores.  -inf and NaN rank last.
//
// route_kernel: 16 lanes a token, four tokens a wave, lane l holds experts l, l + 16, .. as integers of the values' order, whose
// last 4 (5) bits are the place in the lane.  Each lane sorts its own, and a pick is a maximum over the lanes' first ones
// (lane moves inside the row of 16, DPP).  It ranks fp32 scores, whose error is below 2^-21 (1 + s + |r|) (score32).  Where
// two neighbours of the order are closer than twice that and the last bits (of 256 random experts 1 row in 320 to 640 with a
// bias, in 2300 without one; never for bf16 logits without a bias), the k and the next one are put in the order of their
// float64 values; where that does not settle it, the last group in and the first one out are as close (1 row in 9000, 4 of 8
// groups), or anything is not finite, the whole wave ranks the token in float64 (rank_f64).  The weights are of float64
// scores, of the k picked alone (softmax: the sum over the row is of fp32 exponentials).
// What bounds it is issue and latency: 16384 tokens of 256 experts in 8 groups, k = 8, 17.6-20 us (17.8 MB, 2.9 us of bytes;
// a wave is 1640 vector instructions, four waves a SIMD, which are active for 11 us; 19-22 where each pick searched a lane's
// 16 values, about 85 instructions for four tokens against 35 and 130 for the sort); 1031 tokens of 100, k = 4, 4.1 us; one
// token 4.5 us (three dependent latencies and float64 weights).
// route_f64_kernel: one token a wave in float64 throughout, for what the first does not take (more than 16 columns or 512 experts,
// groups of no whole 16): 16384 tokens of 160 experts in 8 groups, k = 6, 36 us; of 256, k = 16 and a shared one, 64 us; one token
// 6.7 us.
#include "smla_internal.h"

namespace {

struct RouteArgs {
  const void* logits;
  int64_t ld;  // elements between rows
  const float* bias;
  int32_t* ids;
  float* weights;
  int64_t T;
  const int32_t* given;  // [T, k] ids whose weights are asked for, or null
  int E, k, groups, topk_groups, renorm, shared;
  double scale;
};

__device__ inline double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int CTRL>
__device__ inline double dpp_f64(double v) {
  return __hiloint2double(dpp_i<CTRL>(__double2hiint(v)), dpp_i<CTRL>(__double2loint(v)));
}
__device__ inline double readlane_f64(double v, int lane) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}
__device__ inline double wave_max_f64(double v) {  // (lane moves: through LDS, ten steps a pick were most of a token's 10 us)
  v = fmax(v, dpp_f64<0xB1>(v));
  v = fmax(v, dpp_f64<0x4E>(v));
  v = fmax(v, dpp_f64<0x141>(v));
  v = fmax(v, dpp_f64<0x140>(v));
  return fmax(fmax(readlane_f64(v, 0), readlane_f64(v, 16)), fmax(readlane_f64(v, 32), readlane_f64(v, 48)));
}
__device__ inline int wave_min_i(int v) {
  v = min(v, dpp_i<0xB1>(v));
  v = min(v, dpp_i<0x4E>(v));
  v = min(v, dpp_i<0x141>(v));
  v = min(v, dpp_i<0x140>(v));
  return min(min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             min(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

template <int SCORE>
__device__ inline double score_f64(double x) {
  if constexpr (SCORE == SMLA_SCORE_SIGMOID) return 1.0 / (1.0 + exp(-x));
  else return sqrt(fmax(x, 0.0) + log1p(exp(-fabs(x))));
}

constexpr double kOut = -__builtin_inf();  // not in the running

// lane j < k: the j-th id and its score; then the shared experts
__device__ inline void finish_f64(const RouteArgs& a, int64_t t, int id, double w) {
  const int lane = threadIdx.x & 63, n = a.k + a.shared;
  if (a.renorm) {
    const double total = wave_sum_f64(lane < a.k ? w : 0.0);
    w = total > 0 ? w / total : total;  // all 0: 0
  }
  if (lane < n) {
    a.ids[t * n + lane] = lane < a.k ? id : a.E + lane - a.k;
    a.weights[t * n + lane] = lane < a.k ? (float)(w * a.scale) : 1.f;
  }
}

// One token in float64 by the whole wave: lane j < k gets the j-th id and its score.  lds: 128 V doubles.
template <int XDT, int SCORE, int V>
__device__ inline void rank_f64(const RouteArgs& a, int64_t t, double* lds, int& mine, double& w) {
  const int lane = threadIdx.x & 63;
  double s[V], r[V];  // scores; logits
  bool have[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int e = lane + 64 * i;
    have[i] = e < a.E;
    r[i] = have[i] ? load_as_f32(a.logits, t * a.ld + e, XDT) : -SMLA_INF;
  }
  if constexpr (SCORE == SMLA_SCORE_SOFTMAX) {
    double m = r[0];
    bool nan = false;
#pragma unroll
    for (int i = 0; i < V; i++) {
      m = fmax(m, r[i]);
      nan |= r[i] != r[i];
    }
    m = wave_max_f64(m);
    nan = __any(nan);
    double sum = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
      s[i] = m == kOut ? 0.0 : exp(r[i] - m);  // a row of -inf: every score 0
      sum += s[i];
    }
    sum = wave_sum_f64(sum);
#pragma unroll
    for (int i = 0; i < V; i++) s[i] = nan ? __builtin_nan("") : sum > 0 ? s[i] / sum : sum;
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) s[i] = score_f64<SCORE>(r[i]);
  }
  if (a.given) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; i++) lds[lane + 64 * i] = s[i];
    __syncthreads();
    mine = lane < a.k ? a.given[t * a.k + lane] : -1;
    w = mine >= 0 && mine < a.E ? lds[mine] : 0.0;
    return;
  }
  double v[V];
#pragma unroll
  for (int i = 0; i < V; i++) v[i] = a.bias && have[i] ? s[i] + (double)a.bias[lane + 64 * i] : s[i];
  if (a.groups > 1) {
    double *rank = lds, *gv = lds + 64 * V;
    const int per = a.E / a.groups;
    __syncthreads();  // (a workgroup is one wave)
#pragma unroll
    for (int i = 0; i < V; i++)
      if (have[i]) rank[lane + 64 * i] = v[i] != v[i] ? kOut : v[i];
    __syncthreads();
    int each = 1;  // lanes of a group: a power of two
    while (2 * each * a.groups <= 64) each *= 2;
    for (int g0 = 0; g0 < a.groups; g0 += 64 / each) {
      const int g = g0 + lane / each;
      double b0 = kOut, b1 = kOut;
      auto add = [&](double x) {
        b1 = fmax(b1, fmin(b0, x));
        b0 = fmax(b0, x);
      };
      if (g < a.groups)
        for (int j = lane % each; j < per; j += each) add(rank[g * per + j]);
      for (int o = 1; o < each; o *= 2) {
        const double c0 = __shfl_xor(b0, o, 64), c1 = __shfl_xor(b1, o, 64);
        add(c0);
        add(c1);
      }
      const double sum = per > 1 ? b0 + b1 : b0;
      if (g < a.groups && lane % each == 0) gv[g] = sum != sum ? kOut : sum;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; i++) {
      if (!have[i]) continue;
      const int g = (lane + 64 * i) / per;
      int before = 0;  // groups ahead of this one
      for (int o = 0; o < a.groups; o++) before += gv[o] > gv[g] || (gv[o] == gv[g] && o < g);
      if (before >= a.topk_groups) have[i] = false;
    }
  }
  bool low[V];  // in the running, but -inf or NaN
#pragma unroll
  for (int i = 0; i < V; i++) {
    if (!a.bias) v[i] = r[i];
    low[i] = have[i] && !(v[i] > kOut);
    if (!have[i] || low[i]) v[i] = kOut;
  }
  mine = -1, w = 0;
  for (int j = 0; j < a.k; j++) {
    double top = v[0];
#pragma unroll
    for (int i = 1; i < V; i++) top = fmax(top, v[i]);
    top = wave_max_f64(top);
    int id = 0x7fffffff;
#pragma unroll
    for (int i = V - 1; i >= 0; i--)
      if (top == kOut ? low[i] : v[i] == top) id = lane + 64 * i;
    id = wave_min_i(id);
    double sj = 0;
#pragma unroll
    for (int i = 0; i < V; i++)
      if (lane + 64 * i == id) {
        v[i] = kOut;
        low[i] = false;
        sj = s[i];
      }
    sj = readlane_f64(sj, id & 63);
    if (lane == j) mine = id, w = sj;
  }
}

template <int XDT, int SCORE, int V>
__global__ __launch_bounds__(64) void route_f64_kernel(const RouteArgs a) {
  __shared__ double lds[128 * V];
  int id;
  double w;
  rank_f64<XDT, SCORE, V>(a, blockIdx.x, lds, id, w);
  finish_f64(a, blockIdx.x, id, w);
}

// ---- 16 lanes a token

// row-of-16 reductions, every lane gets the result
template <class F>
__device__ inline float row_reduce(float v, F&& f) {
  v = f(v, dpp_f<0xB1>(v));
  v = f(v, dpp_f<0x4E>(v));
  v = f(v, dpp_f<0x141>(v));
  return f(v, dpp_f<0x140>(v));
}
__device__ inline float row_max(float v) { return row_reduce(v, [](float x, float y) { return fmaxf(x, y); }); }
template <class F>
__device__ inline int row_reduce_i(int v, F&& f) {
  v = f(v, dpp_i<0xB1>(v));
  v = f(v, dpp_i<0x4E>(v));
  v = f(v, dpp_i<0x141>(v));
  return f(v, dpp_i<0x140>(v));
}
__device__ inline int row_max_i(int v) { return row_reduce_i(v, [](int x, int y) { return max(x, y); }); }
__device__ inline int row_min_i(int v) { return row_reduce_i(v, [](int x, int y) { return min(x, y); }); }

// a float as an integer of the same order (-0 as 0; no NaN): integer maxima need no care for NaN and take their operand from
// another lane as they are
__device__ inline int to_key(float x) {
  const int b = __float_as_int(x + 0.f);
  return b ^ (b >> 31 & 0x7fffffff);
}
__device__ inline float of_key(int k) { return __int_as_float(k ^ (k >> 31 & 0x7fffffff)); }
constexpr int kOutKey = -0x7fffffff - 1, kLowKey = (int)0x807fffff;  // not in the running; -inf
__device__ inline double row_sum_f64(double v) {
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) v += __shfl_xor(v, o, 16);
  return v;
}

// fp32 score, off by less than 2^-21 (1 + s): exp(-|x|) is off by (|x| + 4) 2^-23 of it (the argument's product, the
// instruction), which times its share in s (at most s (1 - s) |x| < 1/4 for the sigmoid, e^(-|x|/2) |x| < 3/4 for the root)
// stays below 2^-22; the quotient, the series and the root add a few 2^-24 of s.
template <int SCORE>
__device__ inline float score32(float x) {
  const float t = __expf(-fabsf(x));
  if constexpr (SCORE == SMLA_SCORE_SIGMOID) {
    return (x >= 0.f ? 1.f : t) * __builtin_amdgcn_rcpf(1.f + t);
  } else {
    // log(1 + t) = 2 (z + z^3 / 3 + z^5 / 5 + ..), z = t / (2 + t) <= 1/3: the first term left out is below 2^-27
    const float z = t * __builtin_amdgcn_rcpf(2.f + t), q = z * z;
    float p = 1.f / 15.f;
    p = fmaf(p, q, 1.f / 13.f);
    p = fmaf(p, q, 1.f / 11.f);
    p = fmaf(p, q, 1.f / 9.f);
    p = fmaf(p, q, 1.f / 7.f);
    p = fmaf(p, q, 1.f / 5.f);
    p = fmaf(p, q, 1.f / 3.f);
    p = fmaf(p, q, 1.f);
    return __builtin_amdgcn_sqrtf(fmaf(2.f * z, p, fmaxf(x, 0.f)));
  }
}

constexpr float kTol = 0x1p-20f;  // twice a score's error

// a lane's keys, largest first (Batcher's odd-even merge sort)
template <int V>
__device__ inline void sort_keys(int (&key)[V]) {
#pragma unroll
  for (int p = 1; p < V; p *= 2)
#pragma unroll
    for (int d = p; d >= 1; d /= 2)
#pragma unroll
      for (int i = 0; i + d < V; i++)
        if (i >= d % p && (i - d % p) / d % 2 == 0 && i / (2 * p) == (i + d) / (2 * p)) {
          const int a = key[i], b = key[i + d];
          key[i] = max(a, b), key[i + d] = min(a, b);
        }
}

template <int XDT, int SCORE, int V>
__global__ __launch_bounds__(64) void route_kernel(const RouteArgs a) {
  constexpr int V64 = (V + 3) / 4;
  __shared__ double lds[128 * V64];
  const int lane = threadIdx.x, l = lane & 15;
  const int64_t t0 = (int64_t)blockIdx.x * 4, row = min(t0 + (lane >> 4), a.T - 1);  // rows past the last repeat it
  const int64_t at = row * a.ld;
  float x[V], v[V];  // logits; ranking values
#pragma unroll
  for (int i = 0; i < V; i++) x[i] = load_as_f32(a.logits, at + min(l + 16 * i, a.E - 1), XDT);
  float b[V];  // (read with the logits; clamped indexes and selects: a guard would put a branch around every load)
  const bool add = a.bias && !a.given;
  if (add) {
#pragma unroll
    for (int i = 0; i < V; i++) b[i] = a.bias[min(l + 16 * i, a.E - 1)];
  }
#pragma unroll
  for (int i = 0; i < V; i++) x[i] = l + 16 * i < a.E ? x[i] : -SMLA_INF;
  bool bad = false;  // this token is ranked in float64
  float m = -SMLA_INF;
  double sum = 1.0;
  if constexpr (SCORE == SMLA_SCORE_SOFTMAX) {
#pragma unroll
    for (int i = 0; i < V; i++) m = fmaxf(m, x[i]);
    m = row_max(m);
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < V; i++) {
      v[i] = expf(x[i] - m);
      sum += v[i];
    }
    sum = row_sum_f64(sum);
    bad = !(sum < SMLA_INF);  // a NaN, an infinite maximum
    const float inv = (float)(1.0 / sum);
#pragma unroll
    for (int i = 0; i < V; i++) v[i] *= inv;
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) bad |= x[i] != x[i];
    if (a.bias || a.groups > 1) {
#pragma unroll
      for (int i = 0; i < V; i++) v[i] = score32<SCORE>(x[i]);
    }
  }
  int mine = -1;
  if (a.given) {
    if (l < a.k) mine = a.given[row * a.k + l];
    bad = __any(bad) && SCORE == SMLA_SCORE_SOFTMAX ? bad : false;  // else each id's score stands alone
  } else {
    float scale = 1.f;  // 1 + the largest score: a bias may take most of one away, but not its error
    if (add) {
      if constexpr (SCORE == SMLA_SCORE_SQRTSOFTPLUS) {  // (the others' are 1 at most)
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < V; i++) s = fmaxf(s, v[i]);
        scale += row_max(s);
      }
#pragma unroll
      for (int i = 0; i < V; i++) {
        v[i] = l + 16 * i < a.E ? v[i] + b[i] : -SMLA_INF;
        bad |= v[i] != v[i];
      }
    }
    int key[V];
#pragma unroll
    for (int i = 0; i < V; i++) key[i] = to_key(a.bias ? v[i] : x[i]);
    if (a.groups > 1) {
      const int spg = a.E / a.groups / 16;  // values a lane holds of a group
      int gv = kOutKey, b0 = gv, b1 = gv;   // lane g: group g's value
      int g = 0, left = spg;
      float parts = 0.f;                    // the magnitudes that its sum is of
#pragma unroll
      for (int i = 0; i < V; i++) {
        const int r = a.bias ? key[i] : to_key(v[i]);
        b1 = max(b1, min(b0, r));
        b0 = max(b0, r);
        if (--left == 0) {  // uniform
          int c0 = b0, c1 = b1;
          auto merge = [&](auto other) __attribute__((always_inline)) {
            const int low = min(c0, other(c0));
            c1 = max(max(c1, other(c1)), low);
            c0 = max(c0, other(c0));
          };
          merge([](int q) { return dpp_i<0xB1>(q); });
          merge([](int q) { return dpp_i<0x4E>(q); });
          merge([](int q) { return dpp_i<0x141>(q); });
          merge([](int q) { return dpp_i<0x140>(q); });
          if (l == g && g < a.groups) {
            gv = to_key(of_key(c0) + of_key(c1));
            parts = gv > kLowKey ? fabsf(of_key(c0)) + fabsf(of_key(c1)) : 0.f;
          }
          g++, left = spg;
          b0 = b1 = kOutKey;
        }
      }
      int before = 0;  // groups ahead of this lane's
#define SMLA_ROR(n) before += dpp_i<0x120 + n>(gv) > gv - (dpp_i<0x120 + n>(l) < l);
      SMLA_ROR(1) SMLA_ROR(2) SMLA_ROR(3) SMLA_ROR(4) SMLA_ROR(5) SMLA_ROR(6) SMLA_ROR(7) SMLA_ROR(8)
      SMLA_ROR(9) SMLA_ROR(10) SMLA_ROR(11) SMLA_ROR(12) SMLA_ROR(13) SMLA_ROR(14) SMLA_ROR(15)
#undef SMLA_ROR
      const bool in = l < a.groups && before < a.topk_groups;
      const int last = row_min_i(in ? gv : 0x7fffffff), next = row_max_i(in ? kOutKey : gv);
      // (a group's value is the sum of two: twice the error)
      if (a.topk_groups < a.groups) bad |= !(of_key(last) - of_key(next) > 2.f * kTol * (scale + row_max(parts))) || last <= kLowKey;
      uint32_t kept = (uint32_t)(__ballot(in) >> (lane & 48)) & 0xffffu;
      left = spg;
#pragma unroll
      for (int i = 0; i < V; i++) {
        if (!(kept & 1)) key[i] = kOutKey;
        if (--left == 0) kept >>= 1, left = spg;
      }
    }
    // A lane's values in order, the place among its 16 (32) instead of the last bits: a pick takes from the lanes' first ones
    constexpr int kPlace = V <= 16 ? 15 : 31;
#pragma unroll
    for (int i = 0; i < V; i++) key[i] = key[i] == kOutKey ? kOutKey : (key[i] & ~kPlace) | (kPlace - i);
    sort_keys<V>(key);
    auto best = [&]() __attribute__((always_inline)) { return row_max_i(key[0]); };
    auto pick = [&](int top, int j) __attribute__((always_inline)) {  // its lowest id to lane j, out of the running
      const int from = row_min_i(key[0] == top ? l : 16);
      const bool pop = l == from;
#pragma unroll
      for (int i = 0; i + 1 < V && i < 16; i++) key[i] = pop ? key[i + 1] : key[i];
      if (V <= 16) key[V - 1] = pop ? kOutKey : key[V - 1];
      if (l == j) mine = (kPlace - (top & kPlace)) * 16 + from;
    };
    // Neighbours in the order that the keys cannot tell apart: the scores' error, and what the last bits were worth
    // (bf16 logits have none there)
    const bool exact = XDT == SMLA_BF16 && !a.bias;
    const float lost = V <= 16 ? 0x1p-18f : 0x1p-17f, tol0 = a.bias ? kTol * scale : 0.f, tol1 = a.bias ? kTol + lost : lost;
    bool close = false;
    float prev = SMLA_INF;
    int top;
    for (int j = 0;; j++) {
      top = best();
      if (!exact) {
        const float now = of_key(top & ~kPlace);
        if (j > 0) close |= !(prev - now > fmaf(tol1, fabsf(prev), tol0)) && top != kOutKey;
        prev = now;
      }
      if (j == a.k) break;
      bad |= (top | kPlace) <= kLowKey;
      pick(top, j);
    }
    if (__any(close)) {
      // the k and the next one in the order of their float64 values, a lane each; the one after it has to be apart
      if ((SCORE != SMLA_SCORE_SOFTMAX || !a.bias) && a.k < 16) {
        pick(top, a.k);
        const int after = best();
        // (prev is the next one's value: what is apart from it is apart from the k-th)
        if (close)
          bad |= (top | kPlace) <= kLowKey || !(prev - of_key(after & ~kPlace) > fmaf(tol1, fabsf(prev), tol0) || after == kOutKey);
        double r = kOut;
        if (l <= a.k && mine < a.E) {
          const float y = load_as_f32(a.logits, at + mine, XDT);
          if constexpr (SCORE == SMLA_SCORE_SOFTMAX) r = y;
          else r = a.bias ? score_f64<SCORE>(y) + (double)a.bias[mine] : y;
        }
        int place = 0;
#pragma unroll
        for (int o = 1; o < 16; o++) {
          const int from = (lane & 48) + ((l + o) & 15), oid = __shfl(mine, from, 64);
          const double other = __shfl(r, from, 64);
          place += ((l + o) & 15) <= a.k && (other > r || (other == r && oid < mine));
        }
        int* ids = (int*)lds;
        if (l <= a.k) ids[(lane & 48) + place] = mine;
        __syncthreads();  // (one wave)
        if (l <= a.k) mine = ids[lane];
      } else {
        bad |= close;
      }
    }
  }
  double w = 0;
  if (l < a.k && mine >= 0 && mine < a.E) {
    const float y = load_as_f32(a.logits, at + mine, XDT);
    if constexpr (SCORE == SMLA_SCORE_SOFTMAX) w = exp((double)y - (double)m) / sum;
    else w = score_f64<SCORE>(y);
  }
  if (a.renorm) {
    const double total = row_sum_f64(l < a.k ? w : 0.0);
    w = total > 0 ? w / total : total;  // all 0: 0
  }
  uint64_t again = __ballot(bad);
  const int n = a.k + a.shared;
  if (l < n && t0 + (lane >> 4) < a.T && !(again >> (lane & 48) & 0xffffu)) {
    a.ids[row * n + l] = l < a.k ? mine : a.E + l - a.k;
    a.weights[row * n + l] = l < a.k ? (float)(w * a.scale) : 1.f;
  }
  while (again) {
    const int g = (__ffsll((unsigned long long)again) - 1) / 16;
    again &= ~(0xffffull << (16 * g));
    const int64_t t = t0 + g;
    if (t >= a.T) break;
    int id;
    double ww;
    rank_f64<XDT, SCORE, V64>(a, t, lds, id, ww);
    finish_f64(a, t, id, ww);
  }
}

template <int XDT, int SCORE>
int launch_route(const RouteArgs& a, hipStream_t st) {
  // 16 lanes a token: up to 32 values a lane, a lane for every group and every column, whole 16s in a group
  const bool rows16 = a.E <= 512 && a.k + a.shared <= 16 &&
                      (a.groups == 1 || a.given || (a.groups <= 16 && a.E / a.groups % 16 == 0));
  const dim3 blk(64), grid((unsigned)(rows16 ? (a.T + 3) / 4 : a.T));
  if (rows16 && a.E <= 64) hipLaunchKernelGGL((route_kernel<XDT, SCORE, 4>), grid, blk, 0, st, a);
  else if (rows16 && a.E <= 128) hipLaunchKernelGGL((route_kernel<XDT, SCORE, 8>), grid, blk, 0, st, a);
  else if (rows16 && a.E <= 256) hipLaunchKernelGGL((route_kernel<XDT, SCORE, 16>), grid, blk, 0, st, a);
  else if (rows16) hipLaunchKernelGGL((route_kernel<XDT, SCORE, 32>), grid, blk, 0, st, a);
  else if (a.E <= 256) hipLaunchKernelGGL((route_f64_kernel<XDT, SCORE, 4>), grid, blk, 0, st, a);
  else hipLaunchKernelGGL((route_f64_kernel<XDT, SCORE, 16>), grid, blk, 0, st, a);
  SMLA_HIP_CHECK_LAUNCH();
  return SMLA_OK;
}

}  // namespace

extern "C" int smla_route(const void* logits, int dtype, int64_t ld, const float* bias, int64_t T, int64_t E, int64_t k, int score,
                          int64_t groups, int64_t topk_groups, int renorm, double scale, int64_t shared, const int32_t* given,
                          int32_t* ids, float* weights, void* stream) {
  if (dtype != SMLA_F32 && dtype != SMLA_BF16) return SMLA_E_DTYPE;
  if (T < 0 || E <= 0 || k <= 0 || groups <= 0 || topk_groups <= 0 || shared < 0 || (T > 1 && ld < E)) return SMLA_E_SHAPE;
  if (score < SMLA_SCORE_SOFTMAX || score > SMLA_SCORE_SQRTSOFTPLUS || !(scale == scale)) return SMLA_E_RANGE;
  if (!given && (E % groups != 0 || topk_groups > groups || k > topk_groups * (E / groups))) return SMLA_E_SHAPE;
  if (E > 1024 || k + shared > 64 || T >= 1 << 26) return SMLA_E_UNSUPPORTED;  // (a grid holds 2^32 threads)
  if (T == 0) return SMLA_OK;
  if (!logits || !ids || !weights) return SMLA_E_NULL;
  const RouteArgs a{logits, ld, bias, ids, weights, T, given, (int)E, (int)k, (int)groups, (int)topk_groups, renorm != 0, (int)shared, scale};
  hipStream_t st = (hipStream_t)stream;
  const bool f = dtype == SMLA_F32;
  switch (score) {
    case SMLA_SCORE_SOFTMAX:
      return f ? launch_route<SMLA_F32, SMLA_SCORE_SOFTMAX>(a, st) : launch_route<SMLA_BF16, SMLA_SCORE_SOFTMAX>(a, st);
    case SMLA_SCORE_SIGMOID:
      return f ? launch_route<SMLA_F32, SMLA_SCORE_SIGMOID>(a, st) : launch_route<SMLA_BF16, SMLA_SCORE_SIGMOID>(a, st);
    default:
      return f ? launch_route<SMLA_F32, SMLA_SCORE_SQRTSOFTPLUS>(a, st) : launch_route<SMLA_BF16, SMLA_SCORE_SQRTSOFTPLUS>(a, st);
  }
}
