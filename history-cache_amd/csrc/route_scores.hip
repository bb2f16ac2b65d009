// Routing of rows to experts by scores, with a bias in the choice and groups of experts, and its gradient:
//
//   s = sigma(l) or softmax(l);  c = s + bias;  a group's rank: the sum of its two largest c;  the top_group best groups stay open
//   chosen: the top_k largest c in open groups, ties to the lowest index;  w = scale * s / (normalize ? sum of the chosen s : 1)
//   S = sum of the chosen s, t = sum_j w[j] g[j]
//   sigmoid:  dl[chosen j] = (normalize ? (scale g[j] - t) / S : scale g[j]) s[j] (1 - s[j])
//   softmax:  dl[chosen j] = w[j] / scale * (scale g[j] - t) (normalize);  dl[e] = p[e] ((e chosen ? scale g : 0) - t)
//
// The bias keeps experts evenly loaded and is no part of the weights; a logit or a bias of -inf closes an expert.  Which of two sums is
// larger is decided in fp64: in fp32 one row in some ten thousand would go to another expert than by the formula.  Without a
// bias experts are compared by their logits, with which the score rises.
//
// A row lies in L lanes, V adjacent logits each, as in route.hip.
#include "route_row.h"

namespace {

constexpr int RS_MAX_GROUPS = 64;
constexpr int RS_SIGMOID = 1;

struct RsArgs {
  const void *logits;
  const float *bias;
  int64_t *expert;
  float *weight, *picked;
  int64_t n;
  float scale;
  int E, k, groups, per_group, top_group;
  bool softmax, normalize, whole;
};

__device__ __forceinline__ int64_t rs_bits(double v) { return __builtin_bit_cast(int64_t, v); }
__device__ __forceinline__ double rs_double(int64_t v) { return __builtin_bit_cast(double, v); }

// ---- fp64 as whole numbers that order like it: NaN above everything, CLOSED below.
constexpr int64_t RS_CLOSED = (int64_t)0x8000000000000000ull;
__device__ __forceinline__ int64_t rs_order(double f) {
  if (f != f) return 0x7fffffffffffffffll;
  if (f == -__builtin_inf()) return RS_CLOSED;
  const int64_t b = rs_bits(f + 0.0);
  return b ^ (b >> 63 & 0x7fffffffffffffffll);
}
__device__ __forceinline__ double rs_value(int64_t o) {
  return o == 0x7fffffffffffffffll ? __builtin_nan("") : rs_double(o ^ (o >> 63 & 0x7fffffffffffffffll));
}

__device__ __forceinline__ double rs_sigma(double l) { return 1.0 / (1.0 + exp(-l)); }

__device__ __forceinline__ int64_t rs_shfl(int64_t v, int lane) {
  const int lo = __shfl((int)(uint32_t)(uint64_t)v, lane, HC_WAVE), hi = __shfl((int)((uint64_t)v >> 32), lane, HC_WAVE);
  return (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
}

// A row's winners, in fp64: winner q * L + lane stays with this lane (-1: none).  row: HC_BLOCK / L rows of L * V numbers in LDS.
template <int L, int V, int KEPT>
__device__ __forceinline__ void rs_choose(const RsArgs &a, const float (&l)[V], int lane, int64_t *row, int (&mine)[KEPT]) {
  const int base = (int)(threadIdx.x & (HC_WAVE - 1)) - lane;
  int64_t key[V];
  double top = -__builtin_inf(), sum = 0.0;
  if (a.softmax) {
    for (int i = 0; i < V; ++i) top = l[i] > top ? (double)l[i] : top;
    top = rs_value(hc_join<L>(rs_order(top), [](int64_t x, int64_t y) { return x > y ? x : y; }));
    for (int i = 0; i < V; ++i) sum += rt_masked(l[i]) ? 0.0 : exp((double)l[i] - top);
    sum = rs_double(hc_join<L>(rs_bits(sum), [](int64_t x, int64_t y) { return rs_bits(rs_double(x) + rs_double(y)); }));
  }
  for (int i = 0; i < V; ++i) {
    const int e = lane * V + i;
    const double s = rt_masked(l[i]) ? 0.0 : a.softmax ? exp((double)l[i] - top) / sum : rs_sigma((double)l[i]);
    const double c = s + (a.bias != nullptr && e < a.E ? (double)a.bias[e] : 0.0);
    row[e] = e >= a.E || rt_masked(l[i]) ? RS_CLOSED : rs_order(c);
    key[i] = a.bias != nullptr || row[e] == RS_CLOSED ? row[e] : rs_order((double)l[i]);
  }
  rt_in_order();
  if (a.groups > 1) {
    constexpr int EACH = RS_MAX_GROUPS / L;
    int64_t rank[EACH];
    for (int u = 0; u < EACH; ++u) {
      const int g = u * L + lane;
      int64_t first = RS_CLOSED, second = RS_CLOSED;
      if (g < a.groups)
        for (int j = 0; j < a.per_group; ++j) {
          const int64_t c = row[g * a.per_group + j];
          second = c > first ? first : c > second ? c : second;
          first = c > first ? c : first;
        }
      rank[u] = second == RS_CLOSED ? first : rs_order(rs_value(first) + rs_value(second));
    }
    uint64_t open = 0;
    for (int u = 0; u < EACH; ++u) {
      const int g = u * L + lane;
      int ahead = 0;
      for (int w = 0; w < EACH; ++w)
        for (int j = 0; j < L; ++j) {
          const int64_t other = rs_shfl(rank[w], base + j);
          const int h = w * L + j;
          if (h < a.groups && (other > rank[u] || (other == rank[u] && h < g))) ++ahead;
        }
      if (g < a.groups && ahead < a.top_group) open |= 1ull << g;
    }
    open = (uint64_t)hc_join<L>((int64_t)open, [](int64_t x, int64_t y) { return x | y; });
    for (int i = 0; i < V; ++i) {
      const int e = lane * V + i;
      if (e < a.E && (open >> (e / a.per_group) & 1) == 0) key[i] = RS_CLOSED;
    }
  }
  for (int q = 0; q < KEPT; ++q) mine[q] = -1;
  for (int j = 0; j < a.k; ++j) {
    int64_t best = key[0];
    int at = lane * V;
    for (int i = 1; i < V; ++i)
      if (key[i] > best) best = key[i], at = lane * V + i;
    const int64_t most = hc_join<L>(best, [](int64_t x, int64_t y) { return x > y ? x : y; });
    const uint32_t won = hc_join<L>(best == most && most != RS_CLOSED ? (uint32_t)at : 0xffffffffu,
                                    [](uint32_t x, uint32_t y) { return x < y ? x : y; });
    for (int i = 0; i < V; ++i)
      if (won == (uint32_t)(lane * V + i)) key[i] = RS_CLOSED;
    for (int q = 0; q < KEPT; ++q)
      if (j == q * L + lane) mine[q] = (int)won;
  }
}

// KEPT: winners a lane keeps, top_k <= KEPT * L.
template <typename T, int L, int V, int KEPT>
__global__ __launch_bounds__(HC_BLOCK) void rs_forward(RsArgs a) {
  __shared__ int64_t s_row[HC_BLOCK * V];
  const int lane = (int)threadIdx.x & (L - 1);
  const int64_t r = ((int64_t)blockIdx.x * HC_BLOCK + threadIdx.x) / L;
  const bool live = r < a.n;
  const auto plus = [](float x, float y) { return x + y; };
  const T *logits = static_cast<const T *>(a.logits) + (live ? r : 0) * a.E;
  T v[V];
  float l[V];
  int mine[KEPT];
  rt_row<T, V>::load(logits, lane * V, a.E, a.whole, v);
#pragma unroll
  for (int i = 0; i < V; ++i) l[i] = hc_to_f32<T>(v[i]);
  rs_choose<L, V, KEPT>(a, l, lane, s_row + (threadIdx.x - lane) * V, mine);
  float top = -__builtin_inff(), all = 0.f;
  if (a.softmax) {
#pragma unroll
    for (int i = 0; i < V; ++i) top = fmaxf(top, l[i]);
    top = hc_join<L>(top, [](float x, float y) { return fmaxf(x, y); });
#pragma unroll
    for (int i = 0; i < V; ++i) all += rt_masked(l[i]) ? 0.f : expf(l[i] - top);
    all = hc_join<L>(all, plus);
  }
  float s[KEPT], p[KEPT], sum = 0.f;
#pragma unroll
  for (int q = 0; q < KEPT; ++q) {
    const bool on = q * L + lane < a.k && mine[q] >= 0;
    p[q] = on ? hc_to_f32<T>(logits[mine[q]]) : 0.f;
    const float e = a.softmax ? expf(p[q] - top) : expf(-fabsf(p[q]));
    s[q] = !on ? 0.f : a.softmax ? e : (p[q] < 0.f ? e : 1.f) / (1.f + e);
    sum += s[q];
  }
  sum = hc_join<L>(sum, plus);
  const float of = a.normalize ? (all != all ? all : sum) : a.softmax ? all : 1.f;
#pragma unroll
  for (int q = 0; q < KEPT; ++q) {
    const int j = q * L + lane;
    if (!live || j >= a.k) continue;
    a.expert[r * a.k + j] = mine[q];
    a.weight[r * a.k + j] = mine[q] < 0 || of == 0.f ? 0.f : a.scale * (s[q] / of);
    if (a.picked != nullptr) a.picked[r * a.k + j] = p[q];
  }
}

struct RsGradArgs {
  const void *logits;
  const int64_t *expert;
  const float *weight, *picked, *g;
  void *grad;
  int64_t n;
  float scale;
  int E, k;
  bool softmax, normalize, whole;
};

template <typename T, int L, int V>
__global__ __launch_bounds__(HC_BLOCK) void rs_backward(RsGradArgs a) {
  // the row in LDS: what its choices bring, each from the lane that has read it; zeros elsewhere
  __shared__ __attribute__((aligned(16))) float s_row[HC_BLOCK * V];
  const int lane = (int)threadIdx.x & (L - 1);
  const int64_t r = ((int64_t)blockIdx.x * HC_BLOCK + threadIdx.x) / L;
  const bool live = r < a.n;
  const int64_t at = (live ? r : 0) * a.k;
  const auto plus = [](float x, float y) { return x + y; };
  const bool by_logit = !a.softmax;
  float *own = s_row + threadIdx.x * V, *row = own - lane * V;
#pragma unroll
  for (int i = 0; i < V; ++i) own[i] = 0.f;
  float t = 0.f, sum = 0.f;
  for (int j = lane; j < a.k; j += L) {
    if (a.expert[at + j] < 0) continue;
    t += a.weight[at + j] * a.g[at + j];
    if (by_logit) {
      const float p = a.picked[at + j], e = expf(-fabsf(p));
      sum += (p < 0.f ? e : 1.f) / (1.f + e);
    }
  }
  t = hc_join<L>(t, plus);
  sum = hc_join<L>(sum, plus);
  rt_in_order();
  for (int j = lane; j < a.k; j += L) {
    const int64_t e = a.expert[at + j];
    if (e < 0 || e >= a.E) continue;
    const float d = a.scale * a.g[at + j];
    float out;
    if (by_logit) {
      const float x = expf(-fabsf(a.picked[at + j])), slope = x / ((1.f + x) * (1.f + x));
      out = !a.normalize ? d * slope : sum == 0.f ? 0.f : (d - t) / sum * slope;
    } else {
      out = a.normalize ? a.weight[at + j] / a.scale * (d - t) : d;
    }
    row[e] = out;
  }
  rt_in_order();
  float out[V];
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = own[i];
  if (a.softmax && !a.normalize) {
    T v[V];
    float p[V], top = -__builtin_inff(), all = 0.f;
    rt_row<T, V>::load(static_cast<const T *>(a.logits) + (live ? r : 0) * a.E, lane * V, a.E, a.whole, v);
#pragma unroll
    for (int i = 0; i < V; ++i) top = fmaxf(top, hc_to_f32<T>(v[i]));
    top = hc_join<L>(top, [](float x, float y) { return fmaxf(x, y); });
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float f = hc_to_f32<T>(v[i]);
      p[i] = rt_masked(f) ? 0.f : expf(f - top);
      all += p[i];
    }
    all = hc_join<L>(all, plus);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (all == 0.f ? 0.f : p[i] / all) * (out[i] - t);
  }
  if (live) rt_row<T, V>::store(static_cast<T *>(a.grad) + r * a.E, lane * V, a.E, a.whole, out);
}

static int rs_sizes(int64_t n, int64_t E, int64_t k, int score, float scale) {
  if (score != 0 && score != RS_SIGMOID) return HC_EINVAL;
  if (!(scale > 0.f) || scale == __builtin_inff()) return HC_EINVAL;
  if (!rt_sizes_ok(n, E, k)) return n >= 0 && E >= 1 && k >= 1 && k <= E ? HC_EUNSUPPORTED : HC_EINVAL;
  return HC_OK;
}

}  // namespace

extern "C" int hc_route_scores(const void *logits, int dtype, int64_t n, int64_t E, int64_t top_k, int score, const float *bias,
                               int64_t num_group, int64_t top_group, int normalize, float scale, int64_t *expert, float *weight,
                               float *picked, void *stream) {
  if (const int rc = rs_sizes(n, E, top_k, score, scale)) return rc;
  HC_REQUIRE(num_group >= 1 && num_group <= E && E % num_group == 0 && top_group >= 1 && top_group <= num_group);
  HC_REQUIRE(top_k <= E / num_group * top_group);
  if (num_group > RS_MAX_GROUPS) return HC_EUNSUPPORTED;
  if (n == 0) return dtype >= HC_F32 && dtype <= HC_BF16 ? HC_OK : HC_EDTYPE;
  HC_REQUIRE(logits && expert && weight);
  return rt_with_type(dtype, [&](auto type) {
    typedef decltype(type) T;
    return rt_with_shape((int)E, [&](auto lanes, auto each) {
      constexpr int L = decltype(lanes)::value, V = decltype(each)::value;
      const int64_t blocks = (n + HC_BLOCK / L - 1) / (HC_BLOCK / L);
      if (!hc_grid_ok(blocks)) return (int)HC_EUNSUPPORTED;
      const RsArgs a{logits, bias, expert, weight, picked, n, scale, (int)E, (int)top_k,
                     // (all groups open: as if there were one)
                     top_group == num_group ? 1 : (int)num_group, (int)(E / num_group), (int)top_group, score != RS_SIGMOID,
                     normalize != 0, rt_row<T, V>::whole(logits, E)};
      const auto kernel = top_k <= L ? rs_forward<T, L, V, 1> : rs_forward<T, L, V, L >= RT_MAX_CHOICES ? 1 : RT_MAX_CHOICES / L>;
      kernel<<<dim3((unsigned)blocks), dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(a);
      return hc_launch_status();
    });
  });
}

extern "C" int hc_route_scores_grad(const void *logits, int dtype, int64_t n, int64_t E, int64_t top_k, int score, int normalize,
                                    float scale, const int64_t *expert, const float *weight, const float *picked,
                                    const float *grad_weight, void *grad_logits, void *stream) {
  if (const int rc = rs_sizes(n, E, top_k, score, scale)) return rc;
  if (n == 0) return dtype >= HC_F32 && dtype <= HC_BF16 ? HC_OK : HC_EDTYPE;
  HC_REQUIRE((score == RS_SIGMOID ? picked != nullptr : logits || normalize) && expert && weight && grad_weight && grad_logits);
  return rt_with_type(dtype, [&](auto type) {
    typedef decltype(type) T;
    return rt_with_shape((int)E, [&](auto lanes, auto each) {
      constexpr int L = decltype(lanes)::value, V = decltype(each)::value;
      const int64_t blocks = (n + HC_BLOCK / L - 1) / (HC_BLOCK / L);
      if (!hc_grid_ok(blocks)) return (int)HC_EUNSUPPORTED;
      const RsGradArgs a{logits, expert, weight, picked, grad_weight, grad_logits, n, scale, (int)E, (int)top_k,
                         score != RS_SIGMOID, normalize != 0,
                         rt_row<T, V>::whole(logits, E) && rt_row<T, V>::whole(grad_logits, E)};
      rs_backward<T, L, V><<<dim3((unsigned)blocks), dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(a);
      return hc_launch_status();
    });
  });
}
