// Routing of rows to experts: softmax over E logits, the top_k largest, their weights, and the gradient.
//
//   m = max_e l[e];  p[e] = exp(l[e] - m) / sum exp(l - m);  chosen: the k largest l, ties to the lowest index
//   weight[j] = p[chosen j] / (normalize ? sum of the chosen p : 1); a logit of -inf is never chosen (-1, weight 0)
//   t = sum_j w[j] g[j];  dl[chosen j] = w[j] (g[j] - t), 0 elsewhere (normalize);  dl[e] = p[e] ((e chosen ? g : 0) - t)
//
// A row lies in L lanes, V adjacent logits each (L = 8 for up to 64 experts), 64 / L rows per wave.  A key orders
// by value and, among equal values, by the lower index: 16-bit logits and an index fit one 32-bit key, whose maximum is
// one instruction; fp32 takes 64 bits.  A lane sorts its keys once; the winners then are, one after the other, the largest of the
// row's first keys, and the lane that had it moves up.  With `normalize` the sum runs over the winners alone, and each lane
// takes the exponential of the winner that it keeps.
// Bound: a lane's sort and the k joins of its row forward (500 009 rows of 64 bf16 logits to four of them: 28 us for 88 MB, with
// the winners joined through LDS and the keys not sorted 42; fp32 logits, whose keys take 64 bits, 43 for 152 MB; of 256 experts to
// eight of them 127 for 304 and 227 for 560).  Backward a row's choices are read once, by its first lanes, and go to
// their places through LDS: 15 us for 96 MB, by memory (read by every lane of the row and looked for among its logits 26; 500 009
// rows of 256, eight of them, 80 and 181).  Small batches are bound by the launch: eight rows 4 us.
#include "hc_common.h"

namespace {

constexpr int RT_MAX_EXPERTS = 1024;
constexpr int RT_MAX_CHOICES = 32;

// ---- ordering keys
// A signed number whose upper half (16 bits; fp32: 32) orders like the logit -- a positive one as it is, of a negative one all but the
// sign turned over, NaN above everything, -0 as 0 -- and whose lower half falls with the index: 8 bits for the place in
// the lane, above them, put in when lanes are compared, the lane.  NONE is below every key.
template <typename T>
struct rt_key {
  typedef int32_t type;
  static constexpr type NONE = (type)0x80000000;
  static constexpr uint32_t INF = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  __device__ __forceinline__ static type order(uint32_t upper) {
    return (type)(upper ^ ((uint32_t)((int32_t)upper >> 31) & 0x7fff0000u));
  }
  template <int V>
  __device__ __forceinline__ static void make(const T (&v)[V], type (&key)[V]) {
    uint32_t odd = 0;                      // is there a NaN or a -0 anywhere?
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t b = __builtin_bit_cast(uint16_t, v[i]);
      key[i] = order(b << 16 | (uint32_t)(V - 1 - i));
      odd |= (b & 0x7fffu) > INF || b == 0x8000u ? 1u : 0u;
    }
    if (__ballot(odd != 0) == 0) return;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t b = __builtin_bit_cast(uint16_t, v[i]);
      if ((b & 0x7fffu) > INF) key[i] = (type)(0x7fff0000u | (uint32_t)(V - 1 - i));
      else if (b == 0x8000u) key[i] = (type)(V - 1 - i);
    }
  }
  __device__ __forceinline__ static uint32_t lower(type k) { return (uint32_t)k & 0xffffu; }
  __device__ __forceinline__ static float value(type k) {
    const uint32_t o = (uint32_t)k & 0xffff0000u;
    if (o == 0x7fff0000u) return __builtin_nanf("");
    return hc_to_f32<T>(__builtin_bit_cast(T, (uint16_t)((uint32_t)order(o) >> 16)));
  }
};
template <>
struct rt_key<float> {
  typedef int64_t type;
  static constexpr type NONE = (type)0x8000000000000000ull;
  __device__ __forceinline__ static uint32_t order(uint32_t b) { return b ^ ((uint32_t)((int32_t)b >> 31) & 0x7fffffffu); }
  template <int V>
  __device__ __forceinline__ static void make(const float (&v)[V], type (&key)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float f = v[i] + 0.0f;
      key[i] = (type)((uint64_t)(f != f ? 0x7fffffffu : order(__float_as_uint(f))) << 32 | (uint32_t)(V - 1 - i));
    }
  }
  __device__ __forceinline__ static uint32_t lower(type k) { return (uint32_t)k; }
  __device__ __forceinline__ static float value(type k) {
    return __uint_as_float(order((uint32_t)((uint64_t)k >> 32)));            // (0x7fffffff is a NaN)
  }
};

// Sorts V keys, the largest first (Batcher's odd-even merge sort).
template <int V, typename K>
__device__ __forceinline__ void rt_sort(K (&a)[V]) {
#pragma unroll
  for (int p = 1; p < V; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < V; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const K x = a[i + j], y = a[i + j + k];
            a[i + j] = x > y ? x : y;
            a[i + j + k] = x > y ? y : x;
          }
}

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
  __device__ __forceinline__ static void load(const T *__restrict__ row, int at, int E, bool whole, T (&v)[V]) {
    if (whole && at + V <= E) {
#pragma unroll
      for (int q = 0; q < V; q += PIECE) {
        typename hc_vec<T, PIECE>::U u;
        u.raw = *reinterpret_cast<const typename hc_vec<T, PIECE>::raw_t *>(row + at + q);
#pragma unroll
        for (int i = 0; i < PIECE; ++i) v[q + i] = u.e[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = at + i < E ? row[at + i] : hc_from_f32<T>(-__builtin_inff());
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

// KEPT: winners a lane keeps, top_k <= KEPT * L.
template <typename T, int L, int V, int KEPT>
__global__ __launch_bounds__(HC_BLOCK) void rt_forward(const T *__restrict__ logits, int64_t *__restrict__ expert,
                                                        float *__restrict__ weight, int64_t n, int E, int k, bool normalize,
                                                        bool whole) {
  typedef rt_key<T> key;
  typedef typename key::type key_t;
  const int lane = (int)threadIdx.x & (L - 1);
  const int64_t r = ((int64_t)blockIdx.x * HC_BLOCK + threadIdx.x) / L;
  const bool live = r < n;
  const auto larger = [](key_t a, key_t b) { return a > b ? a : b; };
  const auto plus = [](float a, float b) { return a + b; };
  T v[V];
  key_t have[V], mine[KEPT], top = key::NONE;
  const key_t place = (key_t)(L - 1 - lane) << 8;
  rt_row<T, V>::load(logits + (live ? r : 0) * E, lane * V, E, whole, v);
  key::make(v, have);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (lane * V + i >= E) have[i] = key::NONE;
  rt_sort(have);
#pragma unroll
  for (int q = 0; q < KEPT; ++q) mine[q] = key::NONE;
  for (int j = 0; j < k; ++j) {
    const key_t own = have[0] | place, best = hc_join<L>(own, larger);
    if (j == 0) top = best;
    // (by bits: a choice between neighbours becomes a search for the chosen index)
    const key_t won = own == best ? -1 : 0;
#pragma unroll
    for (int i = 0; i < V; ++i) have[i] = (have[i] & ~won) | ((i + 1 < V ? have[i + 1] : key::NONE) & won);
#pragma unroll
    for (int q = 0; q < KEPT; ++q)
      if (j == q * L + lane) mine[q] = best;
  }
  const float largest = key::value(top);
  float e[KEPT], sum = 0.f;
#pragma unroll
  for (int q = 0; q < KEPT; ++q) {
    const float f = key::value(mine[q]);
    e[q] = q * L + lane >= k || rt_masked(f) ? 0.f : expf(f - largest);
    sum += e[q];
  }
  if (!normalize) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float f = hc_to_f32<T>(v[i]);
      if (!rt_masked(f)) sum += expf(f - largest);
    }
  }
  sum = hc_join<L>(sum, plus);
#pragma unroll
  for (int q = 0; q < KEPT; ++q)
    if (live && q * L + lane < k) {
      const bool none = rt_masked(key::value(mine[q]));
      const int from = L - 1 - (int)(key::lower(mine[q]) >> 8), at = V - 1 - (int)(key::lower(mine[q]) & 0xffu);
      expert[r * k + q * L + lane] = none ? -1 : from * V + at;
      weight[r * k + q * L + lane] = none ? 0.f : e[q] / sum;
    }
}

// What the wave's lanes have written to LDS is what they read from here on (its accesses stay in order, so that only the
// compiler has to keep it).
__device__ __forceinline__ void rt_in_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <typename T, int L, int V>
__global__ __launch_bounds__(HC_BLOCK) void rt_backward(const T *__restrict__ logits, const int64_t *__restrict__ expert,
                                                         const float *__restrict__ weight, const float *__restrict__ g,
                                                         T *__restrict__ grad, int64_t n, int E, int k, bool normalize,
                                                         bool whole) {
  // the row in LDS: what its choices bring, each from the lane that has read it; zeros elsewhere
  __shared__ __attribute__((aligned(16))) float s_row[HC_BLOCK * V];
  const int lane = (int)threadIdx.x & (L - 1);
  const int64_t r = ((int64_t)blockIdx.x * HC_BLOCK + threadIdx.x) / L;
  const bool live = r < n;
  const int64_t at = (live ? r : 0) * k;
  const auto plus = [](float a, float b) { return a + b; };
  const auto larger = [](float a, float b) { return fmaxf(a, b); };
  float *own = s_row + threadIdx.x * V, *row = own - lane * V;
#pragma unroll
  for (int i = 0; i < V; ++i) own[i] = 0.f;
  int64_t e = -1;
  float w = 0.f, d = 0.f, t = 0.f;
  if (lane < k) e = expert[at + lane], w = weight[at + lane], d = g[at + lane];
  if (e >= 0) t = w * d;
  for (int j = lane + L; j < k; j += L)
    if (expert[at + j] >= 0) t += weight[at + j] * g[at + j];
  t = hc_join<L>(t, plus);
  const auto bring = [&](int64_t e, float w, float d) {
    if (e >= 0 && e < E) row[e] = normalize ? w * (d - t) : d;
  };
  rt_in_order();
  bring(e, w, d);
  for (int j = lane + L; j < k; j += L) bring(expert[at + j], weight[at + j], g[at + j]);
  rt_in_order();
  float out[V];
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = own[i];
  if (!normalize) {
    T v[V];
    float p[V], top = -__builtin_inff(), sum = 0.f;
    rt_row<T, V>::load(logits + (live ? r : 0) * E, lane * V, E, whole, v);
#pragma unroll
    for (int i = 0; i < V; ++i) top = fmaxf(top, hc_to_f32<T>(v[i]));
    top = hc_join<L>(top, larger);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float f = hc_to_f32<T>(v[i]);
      p[i] = rt_masked(f) ? 0.f : expf(f - top);
      sum += p[i];
    }
    sum = hc_join<L>(sum, plus);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      p[i] = sum == 0.f ? 0.f : p[i] / sum;
      out[i] = p[i] * (out[i] - t);
    }
  }
  if (live) rt_row<T, V>::store(grad + r * E, lane * V, E, whole, out);
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
      const auto kernel = top_k <= L ? rt_forward<T, L, V, 1> : rt_forward<T, L, V, L >= RT_MAX_CHOICES ? 1 : RT_MAX_CHOICES / L>;
      kernel<<<dim3((unsigned)blocks), dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(
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
