// Rows of logits in registers: keys that order them, their sort, pieces of rows, and the shapes of the routing kernels.
#pragma once

#include "hc_common.h"

#ifdef __HIPCC__

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

// Sorts V keys, the largest first (Batcher's odd-even merge sort); in_order(x, y) leaves the larger one in x.
template <int V, typename K, typename F>
__device__ __forceinline__ void rt_sort(K (&a)[V], F &&in_order) {
#pragma unroll
  for (int p = 1; p < V; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < V; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) in_order(a[i + j], a[i + j + k]);
}

template <int V, typename K>
__device__ __forceinline__ void rt_sort(K (&a)[V]) {
  rt_sort(a, [](K &first, K &second) {
    const K x = first, y = second;
    first = x > y ? x : y;
    second = x > y ? y : x;
  });
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

// What the wave's lanes have written to LDS is what they read from here on (its accesses stay in order, so that only the
// compiler has to keep it).
__device__ __forceinline__ void rt_in_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
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

#endif  // __HIPCC__
