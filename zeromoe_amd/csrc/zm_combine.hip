// zm_combine.hip -- the weighted sum of the experts' rows with its gradient, and the gradient of the routing.
//
//   out[s] = residual[s] + sum_k weights[s][k] y[s][k]
//   dweights[s][k] = <dout[s], y[s][k]>,  dy[s][k] = weights[s][k] dout[s]
//
// and, behind them, the gradient of the weights by the router's logits (zm_router's weights for a fixed selection):
//   p = gate(logits + logit_bias),  c = weights_scale (1 where that is 0)
//   weights[k] = c p[e_k] / N,  N = max(sum_j p[e_j], 2^-14) where weights are normalised, else 1
//   d_k = c dweights[k], less c sum_j dweights[j] p[e_j] / N where N is the sum; all over N
//   g[e] = sum of d_k over the k with e_k = e, plus dprobs[e]
//   softmax: dlogits = p (g - sum_e p g);  sigmoid: g sigmoid(z) sigmoid(-z);  sqrt-softplus: g sigmoid(z) / (2 p)
// Routes with a negative id take no part: their row of y is not read.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/zeromoe.h"
#include "zm_host.hpp"
#include "zm_linear.hpp"

using namespace zm;

namespace {

struct CombineArgs {
  const float *y;         // [S][K][H], strides y_tok and y_route
  const float *weights;   // [S][K]
  const int32_t *ids;     // [S][K] or null
  const float *residual;  // [S][H] or null
  const float *dout;      // [S][H]
  float *out;             // [S][H]
  float *dweights;        // [S][K] or null
  float *dy;              // [S][K][H] contiguous or null
  int64_t y_tok, y_route;
  int64_t S;
  int K, H;
};

template <int V>
struct Vec;
template <>
struct Vec<4> {
  typedef v4f type;
};
template <>
struct Vec<1> {
  typedef float type;
};
template <int V>
__device__ __forceinline__ typename Vec<V>::type vload(const float *p) {
  return *reinterpret_cast<const typename Vec<V>::type *>(p);
}

constexpr int CMB_K = 64;  // routes of a token at most

// A thread sums V columns of one token over its routes; memory bound, the routes' loads go out eight at a time.
template <int V>
__global__ __launch_bounds__(256) void k_combine_rows(CombineArgs g) {
  typedef typename Vec<V>::type F;
  const int64_t s = blockIdx.x;
  const int h = ((int)blockIdx.y * 256 + (int)threadIdx.x) * V;
  if (h >= g.H) return;
  const float *y = g.y + s * g.y_tok + h;
  F acc = g.residual ? vload<V>(g.residual + s * g.H + h) : F{};
  for (int k0 = 0; k0 < g.K; k0 += 8) {
    F v[8];
    float w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool on = k0 + k < g.K && (!g.ids || g.ids[s * g.K + k0 + k] >= 0);
      w[k] = on ? g.weights[s * g.K + k0 + k] : 0.f;
      v[k] = on ? vload<V>(y + (k0 + k) * g.y_route) : F{};
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) acc += w[k] * v[k];
  }
  *reinterpret_cast<F *>(g.out + s * g.H + h) = acc;
}

// One wave per route: the dot product over H, and the route's row of dy.
template <int V>
__global__ __launch_bounds__(256) void k_combine_backward(CombineArgs g) {
  typedef typename Vec<V>::type F;
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= g.S * g.K) return;
  const int64_t s = r / g.K;
  const int k = (int)(r - s * g.K);
  const bool on = !g.ids || g.ids[r] >= 0;
  const float *d = g.dout + s * g.H, *y = g.y + s * g.y_tok + k * g.y_route;
  if (g.dweights) {
    F acc{};
    if (on)
      for (int h = lane * V; h < g.H; h += 64 * V) acc += vload<V>(d + h) * vload<V>(y + h);
    float sum;
    if constexpr (V == 4) sum = (acc.x + acc.y) + (acc.z + acc.w);
    else sum = acc;
    sum = group_sum<64>(sum);
    if (!lane) g.dweights[r] = sum;
  }
  if (g.dy) {
    const float w = on ? g.weights[r] : 0.f;
    for (int h = lane * V; h < g.H; h += 64 * V)
      *reinterpret_cast<F *>(g.dy + r * g.H + h) = on ? w * vload<V>(d + h) : F{};
  }
}

// ============================================================ gradient of the routing

struct RouteGradArgs {
  const float *logits;      // [S][E]
  const float *logit_bias;  // [E] or null
  const int32_t *ids;       // [S][K]
  const float *dweights;    // [S][K]
  const float *dprobs;      // [E] or null
  float *dlogits;           // [S][E]
  int64_t S;
  int E, K, gating, norm;
  float scale;
};

// One wave per token; expert e = lane + 64 i is register i of its lane (E <= 64 P), route k is lane k (K <= 64).
constexpr int ROUTE_WAVES = 4;
template <int P>
__global__ __launch_bounds__(64 * ROUTE_WAVES) void k_router_backward(RouteGradArgs g) {
  __shared__ float prob[ROUTE_WAVES][64 * P];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t s = (int64_t)blockIdx.x * ROUTE_WAVES + wave;
  if (s >= g.S) return;
  const float INF = __builtin_inff();
  // everything the token needs is asked for at once: a memory latency is most of this kernel's time
  float z[P], p[P], u[P], gr[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int e = lane + 64 * i;
    z[i] = e < g.E ? g.logits[s * g.E + e] : -INF;
    p[i] = g.logit_bias && e < g.E ? g.logit_bias[e] : 0.f;
    gr[i] = g.dprobs && e < g.E ? g.dprobs[e] : 0.f;
  }
  const int id = lane < g.K ? g.ids[s * g.K + lane] : -1;
  float d = lane < g.K ? g.dweights[s * g.K + lane] : 0.f;
  d = id >= 0 ? d : 0.f;
  float *out = g.dlogits + s * g.E;
  const bool any = __ballot(id >= 0) != 0, bad = __ballot(id >= g.E) != 0;
  if (!any || bad) {  // a skipped row has no gradient; an id that does not exist has none that could be told
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (lane + 64 * i < g.E) out[lane + 64 * i] = bad ? __builtin_nanf("") : 0.f;
    return;
  }
  float mx = -INF, p_most = 0.f;  // p_most: softmax's largest probability, that of z = mx
#pragma unroll
  for (int i = 0; i < P; ++i) {
    z[i] += p[i];
    mx = fmaxf(mx, z[i]);
  }
  if (g.gating == 0) {
    mx = wave_max(mx);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      p[i] = mx == -INF && z[i] == z[i] ? 0.f : expf(z[i] - mx);  // all -inf: no probability, no gradient
      sum += lane + 64 * i < g.E ? p[i] : 0.f;
    }
    sum = group_sum<64>(sum);
    const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
    p_most = inv;
#pragma unroll
    for (int i = 0; i < P; ++i) p[i] *= inv;
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float a = z[i];
      const float e = expf(-fabsf(a)), r = 1.0f / (1.0f + e), q = a < 0.f ? e * r : r;  // q: sigmoid
      if (g.gating == 1) {
        p[i] = q;
        u[i] = e * r * r;  // (p (1 - p) has no digits left where p is near 1)
      } else {
        // far below zero softplus(z) is e^z to within f32, and its square root's slope half of that root
        p[i] = a < -17.f ? expf(0.5f * a) : sqrtf(fmaxf(a, 0.f) + log1pf(e));
        u[i] = a < -17.f ? 0.5f * p[i] : q / (2.0f * p[i]);
      }
    }
  }
  // the chosen experts' probabilities, in the lanes of their routes
#pragma unroll
  for (int i = 0; i < P; ++i) prob[wave][lane + 64 * i] = p[i];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const float pk = id >= 0 ? prob[wave][id] : 0.f;
  d *= g.scale;
  bool flat = false;  // the weights' sum is constant: sum_e p g is 0 over the routes
  if (g.norm) {
    const float total = group_sum<64>(pk);
    flat = !(total < 6.103515625e-5f);
    float N = 6.103515625e-5f, dot = 0.f;
    if (flat) {
      // Taking one route's d off all of them changes nothing here.  That of the largest p is taken: its own result, a
      // difference of two nearly equal numbers where it is most of the sum (and 0 where it is all of it), is then made
      // of the other routes alone.
      const float top = wave_max(id >= 0 ? pk : -INF);  // (by all lanes, whether they have a route or not)
      const uint64_t valid = __ballot(id >= 0), largest = __ballot(id >= 0 && pk == top);
      const float d0 = readlane_f(d, __builtin_ctzll(largest ? largest : valid));
      d = id >= 0 ? d - d0 : 0.f;
      dot = group_sum<64>(d * pk);
      N = total;
    }
    d = id >= 0 ? (d - dot / N) / N : 0.f;
  }
  // softmax: g - sum p g.  Where one p is more than half of the row, its g is taken off all of them first (sum p is 1),
  // for the same reason; with no such p the sum of two nearly equal numbers does not arise.
  auto centre = [&] {
    if (p_most > 0.5f) {
      float r = 0.f;
      bool here = false;
#pragma unroll
      for (int i = 0; i < P; ++i)
        if (z[i] == mx) r = gr[i], here = true;
      r = readlane_f(r, __builtin_ctzll(__ballot(here)));
#pragma unroll
      for (int i = 0; i < P; ++i) gr[i] -= r;
    }
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) dot += p[i] * gr[i];
    dot = group_sum<64>(dot);
#pragma unroll
    for (int i = 0; i < P; ++i) gr[i] -= dot;
  };
  if (g.gating == 0 && flat && g.dprobs) centre();
  for (int k = 0; k < g.K; ++k) {  // in order: an expert named twice gets both
    const int ek = __builtin_amdgcn_readlane(id, k);
    const float dk = readlane_f(d, k);
#pragma unroll
    for (int i = 0; i < P; ++i) gr[i] += ek == lane + 64 * i ? dk : 0.f;
  }
  if (g.gating == 0) {
    if (!flat) centre();
#pragma unroll
    for (int i = 0; i < P; ++i) gr[i] *= p[i];
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) gr[i] *= u[i];
  }
#pragma unroll
  for (int i = 0; i < P; ++i)
    if (lane + 64 * i < g.E) out[lane + 64 * i] = gr[i];
}

bool quad(const void *p) { return !((uintptr_t)p & 15); }

int check_combine(const char *who, const float *y, int64_t y_tok, int64_t y_route, int64_t S, int K, int H) {
  if (S < 0 || K <= 0 || K > CMB_K || H <= 0) return fail("%s: S >= 0, 1 <= K <= %d and H > 0 are needed", who, CMB_K);
  if (S >= (1 << 24) || S * K >= (1 << 26) || H > (1 << 26))  // 2^32 threads of a launch
    return fail("%s: too large for one launch", who);
  if (y_tok < 0 || y_route < 0) return fail("%s: negative stride", who);
  if (S && !y) return fail("%s: null pointer", who);
  return 0;
}

}  // namespace

extern "C" {

int zm_combine(const float *y, int64_t y_tok, int64_t y_route, const float *weights, const int32_t *ids,
               const float *residual, int64_t S, int K, int H, float *out, void *stream) {
  if (check_combine("zm_combine", y, y_tok, y_route, S, K, H)) return -1;
  if (!S) return 0;
  if (!weights || !out) return fail("zm_combine: null pointer");
  CombineArgs g{};
  g.y = y;
  g.y_tok = y_tok;
  g.y_route = y_route;
  g.weights = weights;
  g.ids = ids;
  g.residual = residual;
  g.out = out;
  g.S = S;
  g.K = K;
  g.H = H;
  const bool vec = !(H & 3) && !(y_tok & 3) && !(y_route & 3) && quad(y) && quad(out) && (!residual || quad(residual));
  const int per = vec ? 1024 : 256;
  const dim3 grid((unsigned)S, (unsigned)((H + per - 1) / per));
  if (grid.y > 65535) return fail("zm_combine: H too large for one launch");
  if (vec) hipLaunchKernelGGL((k_combine_rows<4>), grid, dim3(256), 0, (hipStream_t)stream, g);
  else hipLaunchKernelGGL((k_combine_rows<1>), grid, dim3(256), 0, (hipStream_t)stream, g);
  HIP_OK(hipGetLastError());
  return 0;
}

int zm_combine_backward(const float *dout, const float *y, int64_t y_tok, int64_t y_route, const float *weights,
                        const int32_t *ids, int64_t S, int K, int H, float *dweights, float *dy, void *stream) {
  if (check_combine("zm_combine_backward", dweights ? y : dout, y_tok, y_route, S, K, H)) return -1;
  if (!S || (!dweights && !dy)) return 0;
  if (!dout || (dy && !weights)) return fail("zm_combine_backward: null pointer");
  CombineArgs g{};
  g.dout = dout;
  g.y = y;
  g.y_tok = y_tok;
  g.y_route = y_route;
  g.weights = weights;
  g.ids = ids;
  g.dweights = dweights;
  g.dy = dy;
  g.S = S;
  g.K = K;
  g.H = H;
  const bool vec = !(H & 3) && quad(dout) && (!dweights || (!(y_tok & 3) && !(y_route & 3) && quad(y))) &&
                   (!dy || quad(dy));
  const dim3 grid((unsigned)((S * K + 3) / 4));
  if (vec) hipLaunchKernelGGL((k_combine_backward<4>), grid, dim3(256), 0, (hipStream_t)stream, g);
  else hipLaunchKernelGGL((k_combine_backward<1>), grid, dim3(256), 0, (hipStream_t)stream, g);
  HIP_OK(hipGetLastError());
  return 0;
}

int zm_router_backward(const zm_router_spec *spec, const float *logits, const float *logit_bias, const int32_t *ids,
                       const float *dweights, const float *dprobs, int S, float *dlogits, void *stream) {
  if (!spec) return fail("zm_router_backward: null argument");
  if (spec->n_experts <= 0 || spec->n_experts > 1024) return fail("zm_router_backward: n_experts out of range");
  if (spec->topk <= 0 || spec->topk > 64 || spec->topk > spec->n_experts) return fail("zm_router_backward: bad topk");
  if (spec->gating < 0 || spec->gating > 2) return fail("zm_router_backward: bad gating");
  if (S < 0 || S >= (1 << 26)) return fail("zm_router_backward: S out of range");
  if (!S) return 0;
  if (!logits || !ids || !dweights || !dlogits) return fail("zm_router_backward: null argument");
  RouteGradArgs g{};
  g.logits = logits;
  g.logit_bias = logit_bias;
  g.ids = ids;
  g.dweights = dweights;
  g.dprobs = dprobs;
  g.dlogits = dlogits;
  g.S = S;
  g.E = spec->n_experts;
  g.K = spec->topk;
  g.gating = spec->gating;
  g.norm = spec->weights_norm;
  g.scale = spec->weights_scale != 0.f ? spec->weights_scale : 1.f;
  const dim3 grid((unsigned)(((int64_t)S + ROUTE_WAVES - 1) / ROUTE_WAVES)), b(64 * ROUTE_WAVES);
  const hipStream_t st = (hipStream_t)stream;
  if (g.E <= 64) hipLaunchKernelGGL((k_router_backward<1>), grid, b, 0, st, g);
  else if (g.E <= 128) hipLaunchKernelGGL((k_router_backward<2>), grid, b, 0, st, g);
  else if (g.E <= 256) hipLaunchKernelGGL((k_router_backward<4>), grid, b, 0, st, g);
  else if (g.E <= 512) hipLaunchKernelGGL((k_router_backward<8>), grid, b, 0, st, g);
  else hipLaunchKernelGGL((k_router_backward<16>), grid, b, 0, st, g);
  HIP_OK(hipGetLastError());
  return 0;
}

}  // extern "C"
