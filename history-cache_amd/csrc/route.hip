// Routing of rows to experts: softmax over E logits, the top_k largest, their weights, and the gradient.
//
//   m = max_e l[e];  p[e] = exp(l[e] - m) / sum exp(l - m);  chosen: the k largest l, ties to the lowest index
//   weight[j] = p[chosen j] / (normalize ? sum of the chosen p : 1); a logit of -inf is never chosen (-1, weight 0)
//   t = sum_j w[j] g[j];  dl[chosen j] = w[j] (g[j] - t), 0 elsewhere (normalize);  dl[e] = p[e] ((e chosen ? g : 0) - t)
//
// A row lies in L lanes, V adjacent logits each (L = 8 for up to 64 experts), 64 / L rows per wave; the k winners are
// found one after the other by a maximum over the lane's keys and then over the row's lanes.  A key orders
// by value and, among equal values, by the lower index: 16-bit logits and an index fit one 32-bit key, whose maximum is
// one instruction; fp32 takes 64 bits.  With `normalize` the sum runs over the winners alone, no other exponential is taken.
#include "hc_common.h"

namespace {

constexpr int RT_MAX_EXPERTS = 1024;
constexpr int RT_MAX_CHOICES = 32;      // four winners a lane where a row lies in eight

// ---- ordering keys: NaN above everything, -0 equal to 0, 0 is below every key
template <typename T>
struct rt_key {
  typedef uint32_t type;
  __device__ __forceinline__ static type make(float v, int index) {
    const float f = v + 0.0f;
    const uint16_t b = __builtin_bit_cast(uint16_t, hc_from_f32<T>(f));      // exact: f came from a T
    const uint16_t o = f != f ? 0xffffu : (b & 0x8000u) ? (uint16_t)~b : (uint16_t)(b | 0x8000u);
    return (uint32_t)o << 16 | (uint32_t)(0xffff - index);
  }
  __device__ __forceinline__ static int index(type k) { return 0xffff - (int)(k & 0xffffu); }
  __device__ __forceinline__ static float value(type k) {
    const uint16_t o = (uint16_t)(k >> 16);
    if (o == 0xffffu) return __builtin_nanf("");
    const uint16_t b = (o & 0x8000u) ? (uint16_t)(o ^ 0x8000u) : (uint16_t)~o;
    return hc_to_f32<T>(__builtin_bit_cast(T, b));
  }
  __device__ __forceinline__ static type other(type k, int d) { return (type)__shfl_xor((int)k, d, HC_WAVE); }
};
template <>
struct rt_key<float> {
  typedef uint64_t type;
  __device__ __forceinline__ static type make(float v, int index) {
    const float f = v + 0.0f;
    const uint32_t b = __float_as_uint(f);
    const uint32_t o = f != f ? 0xffffffffu : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (uint64_t)o << 32 | (uint32_t)(0xffff - index);
  }
  __device__ __forceinline__ static int index(type k) { return 0xffff - (int)(uint32_t)k; }
  __device__ __forceinline__ static float value(type k) {
    const uint32_t o = (uint32_t)(k >> 32);
    if (o == 0xffffffffu) return __builtin_nanf("");
    return __uint_as_float((o & 0x80000000u) ? (o ^ 0x80000000u) : ~o);
  }
  __device__ __forceinline__ static type other(type k, int d) {
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)k, d, HC_WAVE);
    const uint32_t hi = (uint32_t)__shfl_xor((int)(uint32_t)(k >> 32), d, HC_WAVE);
    return (uint64_t)hi << 32 | lo;
  }
};

__device__ __forceinline__ bool rt_masked(float v) { return v == -__builtin_inff(); }

// V adjacent elements of a row in pieces of up to 16 bytes.
template <typename T, int V>
struct rt_row {
  static constexpr int PIECE = V * (int)sizeof(T) <= 16 ? V : 16 / (int)sizeof(T);
  // may they be read and written in whole pieces?
  static bool whole(const void *p, int64_t E) {
    return E % PIECE == 0 && reinterpret_cast<uintptr_t>(p) % (sizeof(T) * PIECE) == 0;
  }
  // columns at, at + 1, ...; behind the row's end: -inf
  __device__ __forceinline__ static void load(const T *__restrict__ row, int at, int E, bool whole, float (&v)[V]) {
    if (whole && at + V <= E) {
#pragma unroll
      for (int q = 0; q < V; q += PIECE) {
        float part[PIECE];
        hc_vec<T, PIECE>::load(row + at + q, part);
#pragma unroll
        for (int i = 0; i < PIECE; ++i) v[q + i] = part[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = at + i < E ? hc_to_f32<T>(row[at + i]) : -__builtin_inff();
    }
  }
  __device__ __forceinline__ static void store(T *__restrict__ row, int at, int E, bool whole, const float (&v)[V]) {
    if (whole && at + V <= E) {
#pragma unroll
      for (int q = 0; q < V; q += PIECE) {
        float part[PIECE];
#pragma unroll
        for (int i = 0; i < PIECE; ++i) part[i] = v[q + i];
        hc_vec<T, PIECE>::store(row + at + q, part);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (at + i < E) row[at + i] = hc_from_f32<T>(v[i]);
    }
  }
};

template <typename T, int L, int V>
__global__ __launch_bounds__(HC_BLOCK) void rt_forward(const T *__restrict__ logits, int64_t *__restrict__ expert,
                                                        float *__restrict__ weight, int64_t n, int E, int k, bool normalize,
                                                        bool whole) {
  typedef rt_key<T> key;
  typedef typename key::type key_t;
  constexpr int KEPT = L >= RT_MAX_CHOICES ? 1 : RT_MAX_CHOICES / L;
  const int lane = (int)threadIdx.x & (L - 1);
  const int64_t r = ((int64_t)blockIdx.x * HC_BLOCK + threadIdx.x) / L;
  const bool live = r < n;
  key_t have[V];
  float v[V], sum = 0.f;
  rt_row<T, V>::load(logits + (live ? r : 0) * E, lane * V, E, whole, v);
#pragma unroll
  for (int i = 0; i < V; ++i) have[i] = lane * V + i < E ? key::make(v[i], lane * V + i) : 0;
  int mine[KEPT];
  float mine_e[KEPT], top = 0.f;
#pragma unroll
  for (int q = 0; q < KEPT; ++q) {
    mine[q] = -1;
    mine_e[q] = 0.f;
  }
  for (int j = 0; j < k; ++j) {
    key_t best = have[0];
#pragma unroll
    for (int i = 1; i < V; ++i) best = have[i] > best ? have[i] : best;
#pragma unroll
    for (int d = L / 2; d >= 1; d /= 2) {
      const key_t o = key::other(best, d);
      best = o > best ? o : best;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) have[i] = have[i] == best ? 0 : have[i];
    const float f = key::value(best);
    if (j == 0) top = f;
    const bool none = rt_masked(f);
    const float e = none ? 0.f : expf(f - top);
    if (normalize) sum += e;
#pragma unroll
    for (int q = 0; q < KEPT; ++q)
      if (j == q * L + lane) {
        mine[q] = none ? -1 : key::index(best);
        mine_e[q] = e;
      }
  }
  if (!normalize) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (!rt_masked(v[i])) sum += expf(v[i] - top);
#pragma unroll
    for (int d = L / 2; d >= 1; d /= 2) sum += __shfl_xor(sum, d, HC_WAVE);
  }
#pragma unroll
  for (int q = 0; q < KEPT; ++q)
    if (live && q * L + lane < k) {
      expert[r * k + q * L + lane] = mine[q];
      weight[r * k + q * L + lane] = mine[q] < 0 ? 0.f : mine_e[q] / sum;
    }
}

template <typename T, int L, int V>
__global__ __launch_bounds__(HC_BLOCK) void rt_backward(const T *__restrict__ logits, const int64_t *__restrict__ expert,
                                                         const float *__restrict__ weight, const float *__restrict__ g,
                                                         T *__restrict__ grad, int64_t n, int E, int k, bool normalize,
                                                         bool whole) {
  const int lane = (int)threadIdx.x & (L - 1);
  const int64_t r = ((int64_t)blockIdx.x * HC_BLOCK + threadIdx.x) / L;
  const bool live = r < n;
  const int64_t at = (live ? r : 0) * k;
  float t = 0.f;
  for (int j = lane; j < k; j += L)
    if (expert[at + j] >= 0) t += weight[at + j] * g[at + j];
#pragma unroll
  for (int d = L / 2; d >= 1; d /= 2) t += __shfl_xor(t, d, HC_WAVE);
  float p[V], out[V];
  if (!normalize) {
    float v[V], top = -__builtin_inff(), sum = 0.f;
    rt_row<T, V>::load(logits + (live ? r : 0) * E, lane * V, E, whole, v);
#pragma unroll
    for (int i = 0; i < V; ++i) top = fmaxf(top, v[i]);
#pragma unroll
    for (int d = L / 2; d >= 1; d /= 2) top = fmaxf(top, __shfl_xor(top, d, HC_WAVE));
#pragma unroll
    for (int i = 0; i < V; ++i) {
      p[i] = rt_masked(v[i]) ? 0.f : expf(v[i] - top);
      sum += p[i];
    }
#pragma unroll
    for (int d = L / 2; d >= 1; d /= 2) sum += __shfl_xor(sum, d, HC_WAVE);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      p[i] = sum == 0.f ? 0.f : p[i] / sum;
      out[i] = -(p[i] * t);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = 0.f;
  }
  for (int j = 0; j < k; ++j) {
    const int64_t e = expert[at + j];
    const float w = weight[at + j], gj = g[at + j];
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (e == lane * V + i) out[i] = (normalize ? w : p[i]) * (gj - t);
  }
  if (!live) return;
  rt_row<T, V>::store(grad + r * E, lane * V, E, whole, out);
}

// L lanes of V logits for E experts, in the first pair that holds them: a row of few experts is spread over eight lanes.
template <typename F>
static int rt_with_shape(int E, F &&f) {
  typedef std::integral_constant<int, 1> c1;
  typedef std::integral_constant<int, 2> c2;
  typedef std::integral_constant<int, 4> c4;
  typedef std::integral_constant<int, 8> c8;
  typedef std::integral_constant<int, 16> c16;
  typedef std::integral_constant<int, 32> c32;
  typedef std::integral_constant<int, 64> c64;
  if (E <= 8) return f(c8{}, c1{});
  if (E <= 16) return f(c8{}, c2{});
  if (E <= 32) return f(c8{}, c4{});
  if (E <= 64) return f(c8{}, c8{});
  if (E <= 128) return f(c16{}, c8{});
  if (E <= 256) return f(c32{}, c8{});
  if (E <= 512) return f(c64{}, c8{});
  return f(c64{}, c16{});
}

template <typename F>
static int rt_with_type(int dtype, F &&f) {
  if (dtype == HC_F32) return f(float{});
  if (dtype == HC_F16) return f(__half{});
  if (dtype == HC_BF16) return f(__hip_bfloat16{});
  return HC_EDTYPE;
}

static bool rt_sizes_ok(int64_t n, int64_t E, int64_t k) {
  return n >= 0 && E >= 1 && E <= RT_MAX_EXPERTS && k >= 1 && k <= RT_MAX_CHOICES && k <= E;
}

}  // namespace

extern "C" int hc_route_rows(const void *logits, int dtype, int64_t n, int64_t E, int64_t top_k, int normalize,
                             int64_t *expert, float *weight, void *stream) {
  if (!rt_sizes_ok(n, E, top_k)) return n >= 0 && E >= 1 && top_k >= 1 && top_k <= E ? HC_EUNSUPPORTED : HC_EINVAL;
  if (n == 0) return dtype >= HC_F32 && dtype <= HC_BF16 ? HC_OK : HC_EDTYPE;
  HC_REQUIRE(logits && expert && weight);
  return rt_with_type(dtype, [&](auto type) {
    typedef decltype(type) T;
    return rt_with_shape((int)E, [&](auto lanes, auto each) {
      constexpr int L = decltype(lanes)::value, V = decltype(each)::value;
      const int64_t blocks = (n + HC_BLOCK / L - 1) / (HC_BLOCK / L);
      if (!hc_grid_ok(blocks)) return (int)HC_EUNSUPPORTED;
      rt_forward<T, L, V><<<dim3((unsigned)blocks), dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(
          static_cast<const T *>(logits), expert, weight, n, (int)E, (int)top_k, normalize != 0,
          rt_row<T, V>::whole(logits, E));
      return hc_launch_status();
    });
  });
}

extern "C" int hc_route_rows_grad(const void *logits, int dtype, int64_t n, int64_t E, int64_t top_k, int normalize,
                                  const int64_t *expert, const float *weight, const float *grad_weight,
                                  void *grad_logits, void *stream) {
  if (!rt_sizes_ok(n, E, top_k)) return n >= 0 && E >= 1 && top_k >= 1 && top_k <= E ? HC_EUNSUPPORTED : HC_EINVAL;
  if (n == 0) return dtype >= HC_F32 && dtype <= HC_BF16 ? HC_OK : HC_EDTYPE;
  HC_REQUIRE((logits || normalize) && expert && weight && grad_weight && grad_logits);
  return rt_with_type(dtype, [&](auto type) {
    typedef decltype(type) T;
    return rt_with_shape((int)E, [&](auto lanes, auto each) {
      constexpr int L = decltype(lanes)::value, V = decltype(each)::value;
      const int64_t blocks = (n + HC_BLOCK / L - 1) / (HC_BLOCK / L);
      if (!hc_grid_ok(blocks)) return (int)HC_EUNSUPPORTED;
      rt_backward<T, L, V><<<dim3((unsigned)blocks), dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(
          static_cast<const T *>(logits), expert, weight, grad_weight, static_cast<T *>(grad_logits), n, (int)E,
          (int)top_k, normalize != 0, rt_row<T, V>::whole(logits, E) && rt_row<T, V>::whole(grad_logits, E));
      return hc_launch_status();
    });
  });
}
