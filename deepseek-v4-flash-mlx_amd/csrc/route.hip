// Routing of tokens to experts (oracle/decode_engine.py:122-128: scores, the balance bias, the top-k, its
// weights), one wave a token.
//
//   s_e = softmax | sigmoid | sqrt(softplus) of the logits;  r_e = s_e + bias_e
//   a group of E / groups experts is worth the sum of its two largest r; the topk_groups best stay
//   ids = the k largest r that stay, in that order; w_j = s[ids_j] (/ their sum) * scale
//
// Ties go to the lowest id, and the order is that of the values and not of their fp32 roundings: two scores an
// fp32 step apart would otherwise trade places with the formula's rounding.  Without a bias the scores' order
// is the logits', which needs no scores.  A NaN ranks below everything.
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
__device__ inline double wave_max_f64(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmax(v, __shfl_xor(v, o, 64));
  return v;
}

template <int SCORE>
__device__ inline double score_of(double x) {
  if constexpr (SCORE == SMLA_SCORE_SIGMOID) return 1.0 / (1.0 + exp(-x));
  else return sqrt(fmax(x, 0.0) + log1p(exp(-fabs(x))));
}

// the largest of the lanes' values v[0 .. V) (id lane + 64 i) and the lowest id that has it; NaN was replaced
template <int V>
__device__ inline int wave_argmax(const double (&v)[V], double& top) {
  const int lane = threadIdx.x & 63;
  double m = v[0];
#pragma unroll
  for (int i = 1; i < V; i++) m = fmax(m, v[i]);
  top = wave_max_f64(m);
  int id = 0x7fffffff;
#pragma unroll
  for (int i = V - 1; i >= 0; i--)
    if (v[i] == top) id = lane + 64 * i;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) id = min(id, __shfl_xor(id, o, 64));
  return id;
}

// lane j < k: the j-th id and its score; then the shared experts
__device__ inline void finish(const RouteArgs& a, int64_t t, int id, double w) {
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

constexpr double kOut = -__builtin_inf();  // not in the running

template <int XDT, int SCORE, int V>
__global__ __launch_bounds__(64) void route_kernel(const RouteArgs a) {
  const int lane = threadIdx.x;
  const int64_t t = blockIdx.x;
  double s[V], r[V];  // scores; ranking values
  bool have[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int e = lane + 64 * i;
    have[i] = e < a.E;
    const float x = have[i] ? load_as_f32(a.logits, t * a.ld + e, XDT) : -SMLA_INF;
    s[i] = x;
  }
  if constexpr (SCORE == SMLA_SCORE_SOFTMAX) {
    double m = s[0];
    bool nan = false;
#pragma unroll
    for (int i = 0; i < V; i++) {
      m = fmax(m, s[i]);
      nan |= s[i] != s[i];
    }
    m = wave_max_f64(m);
    nan = __any(nan);
    double sum = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
      r[i] = s[i];
      s[i] = m == kOut ? 0.0 : exp(s[i] - m);  // a row of -inf: every score 0
      sum += s[i];
    }
    sum = wave_sum_f64(sum);
#pragma unroll
    for (int i = 0; i < V; i++) s[i] = nan ? __builtin_nan("") : sum > 0 ? s[i] / sum : sum;
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) {
      r[i] = s[i];
      s[i] = score_of<SCORE>(s[i]);
    }
  }
  if (a.given) {  // no choice: the weights of these ids (0 outside 0 .. E-1)
    __shared__ double sc[64 * V];
#pragma unroll
    for (int i = 0; i < V; i++) sc[lane + 64 * i] = s[i];
    __syncthreads();
    const int id = lane < a.k ? a.given[t * a.k + lane] : -1;
    finish(a, t, id, id >= 0 && id < a.E ? sc[id] : 0.0);
    return;
  }
  // ranking values; NaN and what does not exist last
  double v[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int e = lane + 64 * i;
    v[i] = a.bias && have[i] ? s[i] + (double)a.bias[e] : s[i];
    if (!a.bias && a.groups == 1) v[i] = r[i];
  }
  __shared__ double gv[1024], rank[1024];
  if (a.groups > 1) {
    const int per = a.E / a.groups;
#pragma unroll
    for (int i = 0; i < V; i++)
      if (have[i]) rank[lane + 64 * i] = v[i] != v[i] ? kOut : v[i];
    __syncthreads();
    for (int g = lane; g < a.groups; g += 64) {
      double b0 = kOut, b1 = kOut;
      for (int j = 0; j < per; j++) {
        const double w = rank[g * per + j];
        if (w > b0) b1 = b0, b0 = w;
        else if (w > b1) b1 = w;
      }
      const double sum = per > 1 ? b0 + b1 : b0;
      gv[g] = sum != sum ? kOut : sum;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int e = lane + 64 * i;
      if (!have[i]) continue;
      const int g = e / per;
      int before = 0;  // groups ahead of this one
      for (int o = 0; o < a.groups; o++) before += gv[o] > gv[g] || (gv[o] == gv[g] && o < g);
      if (!a.bias) v[i] = r[i];
      if (before >= a.topk_groups) have[i] = false;
    }
  }
  // three classes: in the running, NaN or -inf in the running, out
  bool low[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    low[i] = have[i] && !(v[i] > kOut);
    if (!have[i] || low[i]) v[i] = kOut;
  }
  int mine = -1;        // lane j: the j-th id
  double w = 0;
  for (int j = 0; j < a.k; j++) {
    double top;
    int id = wave_argmax<V>(v, top);
    if (top == kOut) {  // only -inf and NaN are left: by id, -inf before NaN
      id = 0x7fffffff;
#pragma unroll
      for (int i = V - 1; i >= 0; i--)
        if (low[i]) id = lane + 64 * i;
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) id = min(id, __shfl_xor(id, o, 64));
    }
    double sj = 0;
#pragma unroll
    for (int i = 0; i < V; i++)
      if (lane + 64 * i == id) {
        v[i] = kOut;
        low[i] = false;
        sj = s[i];
      }
    sj = __shfl(sj, id & 63, 64);
    if (lane == j) mine = id, w = sj;
  }
  finish(a, t, mine, w);
}

template <int XDT, int SCORE>
int launch_route(const RouteArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.T), blk(64);
  if (a.E <= 256) hipLaunchKernelGGL((route_kernel<XDT, SCORE, 4>), grid, blk, 0, st, a);
  else hipLaunchKernelGGL((route_kernel<XDT, SCORE, 16>), grid, blk, 0, st, a);
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
  if (E > 1024 || k + shared > 64 || T > 0x7fffffff) return SMLA_E_UNSUPPORTED;
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
