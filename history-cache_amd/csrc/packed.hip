// Activations kept in 8 bits for the backward pass.  A row's columns are taken in groups of 32, 64 or 128 (the last one may
// be shorter); a group keeps one fp32 scale and a signed byte per element:
//
//   m = max |x|;  scale = m * (1 / 127);  code = rint(x * (1 / m * 127));  x' = code * scale        (|x' - x| <= scale / 2)
//
// each operation rounded to fp32, one division per group.  A group whose m is below 2^-120, where 127 / m leaves fp32, is kept as zeros; one that holds an infinity or a NaN has that
// as its scale and zeros as codes, so that all of it reads back as NaN.  The largest numbers take the largest scale whose
// 127-fold is finite.
//
// The gate of an expert, h = silu(a) b for rows [a | b], keeps its argument this way (hc_gated_pack) and takes from it in
// backward the gradients of a and b and h itself, which the second product's weight gradient needs (hc_gated_grad):
//   s = sigma(a');  da = dh b' s (1 + a' (1 - s));  db = dh a' s;  h' = a' s b'
// Groups do not reach over from a to b.
//
// A lane owns eight adjacent columns; group / 8 lanes share a group.  Bound by memory: one pass over each operand.
#include "hc_common.h"

namespace {

constexpr float PK_SMALLEST = 0x1p-120f;
constexpr float PK_LARGEST_SCALE = 0x1.0204060000000p+121f;      // 127 times the next one leaves fp32
constexpr int PK_EACH = 8;

// Eight adjacent elements, at no more than their own alignment; those behind `valid` read as zeros and are not written.
template <typename T>
struct pk_row {
  struct __attribute__((packed, aligned(alignof(T)))) eight {
    T e[PK_EACH];
  };
  __device__ __forceinline__ static void load(const T *__restrict__ p, int valid, float (&v)[PK_EACH]) {
    if (valid >= PK_EACH) {
      const eight q = *reinterpret_cast<const eight *>(p);
#pragma unroll
      for (int i = 0; i < PK_EACH; ++i) v[i] = hc_to_f32<T>(q.e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < PK_EACH; ++i) v[i] = i < valid ? hc_to_f32<T>(p[i]) : 0.f;
    }
  }
  __device__ __forceinline__ static void store(T *__restrict__ p, int valid, const float (&v)[PK_EACH]) {
    if (valid >= PK_EACH) {
      eight q;
#pragma unroll
      for (int i = 0; i < PK_EACH; ++i) q.e[i] = hc_from_f32<T>(v[i]);
      *reinterpret_cast<eight *>(p) = q;
    } else {
#pragma unroll
      for (int i = 0; i < PK_EACH; ++i)
        if (i < valid) p[i] = hc_from_f32<T>(v[i]);
    }
  }
};

struct __attribute__((packed, aligned(1))) pk_codes {
  int8_t e[PK_EACH];
};

__device__ __forceinline__ void pk_load_codes(const int8_t *__restrict__ p, int valid, float scale, float (&v)[PK_EACH]) {
  if (valid >= PK_EACH) {
    const pk_codes q = *reinterpret_cast<const pk_codes *>(p);
#pragma unroll
    for (int i = 0; i < PK_EACH; ++i) v[i] = (float)q.e[i] * scale;
  } else {
#pragma unroll
    for (int i = 0; i < PK_EACH; ++i) v[i] = i < valid ? (float)p[i] * scale : 0.f;
  }
}

// The scale of the group that L lanes hold, and this lane's codes.  The largest magnitude is found on the bits, where a NaN
// is above infinity and infinity above every number.
template <int L>
__device__ __forceinline__ float pk_encode(const float (&v)[PK_EACH], int8_t *__restrict__ p, int valid) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < PK_EACH; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
#pragma unroll
  for (int d = L / 2; d >= 1; d /= 2) {
    const uint32_t o = (uint32_t)__shfl_xor((int)m, d, HC_WAVE);
    m = o > m ? o : m;
  }
  const float most = __uint_as_float(m);
  const bool zero = most < PK_SMALLEST, bad = m >= 0x7f800000u;
  const float inverse = zero || bad ? 0.f : 1.0f / most * 127.0f;
  pk_codes q;
#pragma unroll
  for (int i = 0; i < PK_EACH; ++i) q.e[i] = bad ? (int8_t)0 : (int8_t)(int)rintf(v[i] * inverse);
  if (valid >= PK_EACH) {
    *reinterpret_cast<pk_codes *>(p) = q;
  } else {
#pragma unroll
    for (int i = 0; i < PK_EACH; ++i)
      if (i < valid) p[i] = q.e[i];
  }
  const float scale = most * (1.0f / 127.0f);
  return zero ? 0.f : !bad && scale > PK_LARGEST_SCALE ? PK_LARGEST_SCALE : scale;
}

// 1 / (1 + exp(-a)), by exp(-|a|), which does not leave fp32 where the result does not.
__device__ __forceinline__ float pk_sigma(float a) {
  const float e = expf(-fabsf(a));
  return (a < 0.f ? e : 1.f) / (1.f + e);
}

struct PkArgs {
  int64_t items;          // groups of all rows
  int F, groups, group;
};

// What a lane works on: its group's row and number, its first column and how many of its eight are in the row.
template <int L>
struct pk_item {
  int64_t row;
  int g, col, valid, lane;
  bool live;
  __device__ __forceinline__ pk_item(const PkArgs &a) {
    const int64_t t = (int64_t)blockIdx.x * HC_BLOCK + threadIdx.x, i = t / L;
    lane = (int)(t % L);
    live = i < a.items;
    row = live ? i / a.groups : 0;
    g = live ? (int)(i - row * a.groups) : 0;
    col = g * (L * PK_EACH) + lane * PK_EACH;
    valid = live ? a.F - col : 0;
  }
};

template <typename T, int L>
__global__ __launch_bounds__(HC_BLOCK) void pk_pack(PkArgs a, const T *__restrict__ x, int8_t *__restrict__ codes,
                                                    float *__restrict__ scale) {
  const pk_item<L> it(a);
  float v[PK_EACH];
  const int64_t at = it.row * a.F + it.col;
  pk_row<T>::load(x + at, it.valid, v);
  const float s = pk_encode<L>(v, codes + at, it.valid);
  if (it.live && it.lane == 0) scale[it.row * a.groups + it.g] = s;
}

template <typename T, int L>
__global__ __launch_bounds__(HC_BLOCK) void pk_unpack(PkArgs a, const int8_t *__restrict__ codes, const float *__restrict__ scale,
                                                      T *__restrict__ x) {
  const pk_item<L> it(a);
  if (!it.live || it.valid <= 0) return;
  float v[PK_EACH];
  const int64_t at = it.row * a.F + it.col;
  pk_load_codes(codes + at, it.valid, scale[it.row * a.groups + it.g], v);
  pk_row<T>::store(x + at, it.valid, v);
}

template <typename T, int L>
__global__ __launch_bounds__(HC_BLOCK) void pk_gated(PkArgs a, const T *__restrict__ x, T *__restrict__ h,
                                                     int8_t *__restrict__ codes, float *__restrict__ scale) {
  const pk_item<L> it(a);
  float va[PK_EACH], vb[PK_EACH], o[PK_EACH];
  const int64_t at = it.row * 2 * a.F + it.col;
  pk_row<T>::load(x + at, it.valid, va);
  pk_row<T>::load(x + at + a.F, it.valid, vb);
#pragma unroll
  for (int i = 0; i < PK_EACH; ++i) o[i] = va[i] * pk_sigma(va[i]) * vb[i];
  if (it.valid > 0) pk_row<T>::store(h + it.row * a.F + it.col, it.valid, o);
  if (codes == nullptr) return;
  const float sa = pk_encode<L>(va, codes + at, it.valid), sb = pk_encode<L>(vb, codes + at + a.F, it.valid);
  if (it.live && it.lane == 0) {
    scale[(it.row * 2) * a.groups + it.g] = sa;
    scale[(it.row * 2 + 1) * a.groups + it.g] = sb;
  }
}

template <typename T, int L>
__global__ __launch_bounds__(HC_BLOCK) void pk_gated_grad(PkArgs a, const int8_t *__restrict__ codes,
                                                          const float *__restrict__ scale, const T *__restrict__ dh,
                                                          T *__restrict__ dx, T *__restrict__ h) {
  const pk_item<L> it(a);
  if (!it.live || it.valid <= 0) return;
  float va[PK_EACH], vb[PK_EACH], g[PK_EACH], o[PK_EACH];
  const int64_t at = it.row * 2 * a.F + it.col;
  pk_load_codes(codes + at, it.valid, scale[(it.row * 2) * a.groups + it.g], va);
  pk_load_codes(codes + at + a.F, it.valid, scale[(it.row * 2 + 1) * a.groups + it.g], vb);
  pk_row<T>::load(dh + it.row * a.F + it.col, it.valid, g);
#pragma unroll
  for (int i = 0; i < PK_EACH; ++i) {
    const float s = pk_sigma(va[i]), silu = va[i] * s;
    o[i] = silu * vb[i];
    const float da = g[i] * vb[i] * (s * (1.f + va[i] * (1.f - s)));
    vb[i] = g[i] * silu;
    va[i] = da;
  }
  pk_row<T>::store(dx + at, it.valid, va);
  pk_row<T>::store(dx + at + a.F, it.valid, vb);
  if (h != nullptr) pk_row<T>::store(h + it.row * a.F + it.col, it.valid, o);
}

static int pk_args(int64_t n, int64_t F, int64_t group, PkArgs *a) {
  if (n < 0 || F < 1) return HC_EINVAL;
  if ((group != 32 && group != 64 && group != 128) || F >= (1 << 30)) return HC_EUNSUPPORTED;
  a->F = (int)F;
  a->group = (int)group;
  a->groups = (int)((F + group - 1) / group);
  a->items = n * a->groups;
  return hc_grid_ok((a->items * (group / PK_EACH) + HC_BLOCK - 1) / HC_BLOCK + 1) ? HC_OK : HC_EUNSUPPORTED;
}

template <typename F>
static int pk_with(int dtype, const PkArgs &a, F &&f) {
  const auto lanes = [&](auto type) {
    if (a.items == 0) return (int)HC_OK;
    const dim3 grid((unsigned)((a.items * (a.group / PK_EACH) + HC_BLOCK - 1) / HC_BLOCK));
    if (a.group == 32) f(type, std::integral_constant<int, 4>{}, grid);
    else if (a.group == 64) f(type, std::integral_constant<int, 8>{}, grid);
    else f(type, std::integral_constant<int, 16>{}, grid);
    return hc_launch_status();
  };
  if (dtype == HC_F32) return lanes(float{});
  if (dtype == HC_F16) return lanes(__half{});
  if (dtype == HC_BF16) return lanes(__hip_bfloat16{});
  return HC_EDTYPE;
}

}  // namespace

extern "C" int hc_pack_rows(const void *x, int dtype, int64_t n, int64_t F, int64_t group, int8_t *codes, float *scale,
                            void *stream) {
  PkArgs a;
  if (const int rc = pk_args(n, F, group, &a)) return rc;
  HC_REQUIRE(n == 0 || (x && codes && scale));
  return pk_with(dtype, a, [&](auto type, auto lanes, dim3 grid) {
    typedef decltype(type) T;
    pk_pack<T, decltype(lanes)::value><<<grid, dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(
        a, static_cast<const T *>(x), codes, scale);
  });
}

extern "C" int hc_unpack_rows(const int8_t *codes, const float *scale, int64_t n, int64_t F, int64_t group, void *x, int dtype,
                              void *stream) {
  PkArgs a;
  if (const int rc = pk_args(n, F, group, &a)) return rc;
  HC_REQUIRE(n == 0 || (x && codes && scale));
  return pk_with(dtype, a, [&](auto type, auto lanes, dim3 grid) {
    typedef decltype(type) T;
    pk_unpack<T, decltype(lanes)::value><<<grid, dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(
        a, codes, scale, static_cast<T *>(x));
  });
}

extern "C" int hc_gated_pack(const void *x, int dtype, int64_t n, int64_t F, int64_t group, void *h, int8_t *codes,
                             float *scale, void *stream) {
  PkArgs a;
  if (const int rc = pk_args(n, F, group, &a)) return rc;
  HC_REQUIRE((codes == nullptr) == (scale == nullptr) && (n == 0 || (x && h)));
  return pk_with(dtype, a, [&](auto type, auto lanes, dim3 grid) {
    typedef decltype(type) T;
    pk_gated<T, decltype(lanes)::value><<<grid, dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(
        a, static_cast<const T *>(x), static_cast<T *>(h), codes, scale);
  });
}

extern "C" int hc_gated_grad(const int8_t *codes, const float *scale, const void *grad_h, int dtype, int64_t n, int64_t F,
                             int64_t group, void *grad_x, void *h, void *stream) {
  PkArgs a;
  if (const int rc = pk_args(n, F, group, &a)) return rc;
  HC_REQUIRE(n == 0 || (codes && scale && grad_h && grad_x));
  return pk_with(dtype, a, [&](auto type, auto lanes, dim3 grid) {
    typedef decltype(type) T;
    pk_gated_grad<T, decltype(lanes)::value><<<grid, dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(
        a, codes, scale, static_cast<const T *>(grad_h), static_cast<T *>(grad_x), static_cast<T *>(h));
  });
}
