// moe_route.hip -- the router of a layer of experts: logits, scores, choice of
// k experts and their weights (the host routing of engine.cu:878-893 with its
// copy of the logits, on the device).
//
//   l = gate x,  s = 1 / (1 + exp(-l)) or softmax(l),  c = s + bias
//   groups: those topk_group of n_group whose two best c have the largest sum
//   ids = the k largest c among the experts of those groups, largest first,
//   the lowest index first among equals;  w = s[ids]
//   renorm: w / (sum w + eps);  then times scale
//
// Which experts are chosen is decided in 64 bits from the products on: fp16
// products are exact there and the order of their sum does not matter (an
// fp32 sum of 2048 products is 1e-7 off, which moves a choice in one token of
// some 1e5), so a token's experts do not depend on the batch around it.
#include "common.h"
#include "cuda_inf_ffn.h"

namespace cia {

constexpr int kRouteMaxE = CIA_MOE_MAX_EXPERTS;
constexpr int kRouteMaxK = CIA_MOE_MAX_TOP_K;

struct RouteArgs {
  const uint16_t* x;      // fp16 [S][H], or null: logits are given
  const uint16_t* gate;   // fp16 [E][H]
  const float* logits_in; // fp32 [S][E]
  const float* bias;      // fp32 [E], or null
  int32_t* ids;
  float* weights;
  float* logits;          // fp32 [S][E], or null
  int S, H, E, k, softmax, n_group, topk_group, renorm;
  float eps, scale;
};

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// one token a workgroup of 256
__global__ __launch_bounds__(256) void k_moe_route(RouteArgs a) {
  __shared__ double lg[kRouteMaxE], ch[kRouteMaxE], gs[kRouteMaxE], red[4];
  __shared__ double top[kRouteMaxK];
  const int s = blockIdx.x, tid = threadIdx.x, w = tid >> 6, l = tid & 63;
  if (a.x) {
    const uint16_t* xr = a.x + (size_t)s * a.H;
    for (int e = w; e < a.E; e += 4) {
      const uint16_t* gr = a.gate + (size_t)e * a.H;
      double acc = 0.0;
      for (int c = l; c < a.H; c += 64) acc += (double)h2f(xr[c]) * (double)h2f(gr[c]);
      acc = wave_sum_f64(acc);
      if (l == 0) lg[e] = acc;
    }
  } else if (tid < a.E) {
    lg[tid] = (double)a.logits_in[(size_t)s * a.E + tid];
  }
  __syncthreads();
  if (a.logits && tid < a.E) a.logits[(size_t)s * a.E + tid] = (float)lg[tid];
  double sc = 0.0;
  if (a.softmax) {
    double m = -__builtin_inf();
    for (int e = 0; e < a.E; e++) m = lg[e] > m || lg[e] != lg[e] ? lg[e] : m;
    const double p = tid < a.E && m > -__builtin_inf() ? exp(lg[tid] - m) : (m != m ? m : 0.0);
    const double ws = wave_sum_f64(tid < a.E ? p : 0.0);
    if (l == 0) red[w] = ws;
    __syncthreads();
    const double sum = red[0] + red[1] + red[2] + red[3];
    sc = sum == 0.0 ? 0.0 : p / sum;
  } else if (tid < a.E) {
    sc = 1.0 / (1.0 + exp(-lg[tid]));
  }
  // a choice that is not a number ranks with the last
  double c = tid < a.E ? sc + (a.bias ? (double)a.bias[tid] : 0.0) : 0.0;
  if (c != c) c = -__builtin_inf();
  if (tid < a.E) ch[tid] = c;
  __syncthreads();
  bool in = tid < a.E;
  if (a.n_group > 1) {
    const int per = a.E / a.n_group;
    if (tid < a.n_group) {
      double b0 = -__builtin_inf(), b1 = b0;
      for (int i = 0; i < per; i++) {
        const double v = ch[tid * per + i];
        if (v > b0) {
          b1 = b0;
          b0 = v;
        } else if (v > b1) {
          b1 = v;
        }
      }
      const double t = per > 1 ? b0 + b1 : b0;
      gs[tid] = t != t ? -__builtin_inf() : t;
    }
    __syncthreads();
    if (in) {
      const int g = tid / per;
      int rank = 0;
      for (int j = 0; j < a.n_group; j++) rank += gs[j] > gs[g] || (gs[j] == gs[g] && j < g);
      in = rank < a.topk_group;
    }
    __syncthreads();
    if (tid < a.E) gs[tid] = in ? 1.0 : 0.0;
    __syncthreads();
  }
  int rank = a.k;
  if (in) {
    rank = 0;
    for (int j = 0; j < a.E; j++)
      if (a.n_group == 1 || gs[j] != 0.0) rank += ch[j] > c || (ch[j] == c && j < tid);
  }
  if (rank < a.k) {
    top[rank] = sc;
    a.ids[(size_t)s * a.k + rank] = tid;
  }
  __syncthreads();
  if (tid < a.k) {
    double f = (double)a.scale;
    if (a.renorm) {
      double sum = (double)a.eps;
      for (int j = 0; j < a.k; j++) sum += top[j];
      f = sum == 0.0 ? 0.0 : f / sum;
    }
    a.weights[(size_t)s * a.k + tid] = (float)(top[tid] * f);
  }
}

static int route_run(const RouteArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(k_moe_route, dim3((unsigned)a.S), dim3(256), 0, s, a);
  return launch_status();
}

// the choice's parameters into a; CIA_ERR_ARG where they contradict each other
static int route_args(RouteArgs& a, const cia_moe_gating* g, int S) {
  CIA_REQUIRE(g, CIA_ERR_NULL);
  CIA_REQUIRE(g->n_experts >= 1 && g->n_experts <= kRouteMaxE && g->top_k >= 1 && g->top_k <= kRouteMaxK &&
                  g->top_k <= g->n_experts && S >= 0,
              CIA_ERR_ARG);
  CIA_REQUIRE(g->score == CIA_SCORE_SIGMOID || g->score == CIA_SCORE_SOFTMAX, CIA_ERR_ARG);
  CIA_REQUIRE(g->n_group >= 1 && g->n_experts % g->n_group == 0 && g->topk_group >= 1 &&
                  g->topk_group <= g->n_group && g->n_experts / g->n_group * g->topk_group >= g->top_k,
              CIA_ERR_ARG);
  CIA_REQUIRE(g->eps >= 0.0f && g->eps < __builtin_inff() && g->scale - g->scale == 0.0f, CIA_ERR_ARG);
  a.S = S;
  a.E = g->n_experts;
  a.k = g->top_k;
  a.softmax = g->score == CIA_SCORE_SOFTMAX;
  a.n_group = g->n_group;
  a.topk_group = g->topk_group;
  a.renorm = g->renorm != 0;
  a.eps = g->eps;
  a.scale = g->scale;
  return CIA_OK;
}

}  // namespace cia

using namespace cia;

extern "C" int cia_moe_route(const uint16_t* x, const uint16_t* gate, const float* bias,
                             const cia_moe_gating* g, int32_t* ids, float* weights, float* logits,
                             int S, int H, void* stream) {
  RouteArgs a{};
  const int st = route_args(a, g, S);
  if (st) return st;
  CIA_REQUIRE(H > 0 && H % 8 == 0, CIA_ERR_ARG);
  if (S == 0) return CIA_OK;
  CIA_REQUIRE(x && gate && ids && weights, CIA_ERR_NULL);
  CIA_REQUIRE(aligned(x, 16) && aligned(gate, 16) && aligned(bias, 4) && aligned(ids, 4) &&
                  aligned(weights, 4) && aligned(logits, 4),
              CIA_ERR_ALIGN);
  a.x = x;
  a.gate = gate;
  a.bias = bias;
  a.ids = ids;
  a.weights = weights;
  a.logits = logits;
  a.H = H;
  return route_run(a, (hipStream_t)stream);
}

extern "C" int cia_moe_select(const float* logits, const float* bias, const cia_moe_gating* g,
                              int32_t* ids, float* weights, int S, void* stream) {
  RouteArgs a{};
  const int st = route_args(a, g, S);
  if (st) return st;
  if (S == 0) return CIA_OK;
  CIA_REQUIRE(logits && ids && weights, CIA_ERR_NULL);
  CIA_REQUIRE(aligned(logits, 4) && aligned(bias, 4) && aligned(ids, 4) && aligned(weights, 4), CIA_ERR_ALIGN);
  a.logits_in = logits;
  a.bias = bias;
  a.ids = ids;
  a.weights = weights;
  return route_run(a, (hipStream_t)stream);
}
