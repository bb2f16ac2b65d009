// Activations kept in 8 bits for the backward pass.  A row's columns are taken in groups of 32, 64 or 128 (the last one may
// be shorter); a group keeps one fp32 scale and a signed byte per element:
//
//   m = max |x|;  scale = m * (1 / 127);  code = rint(x * (1 / m * 127));  x' = code * scale
//
// |x' - x| is at most half a scale and what six fp32 operations on up to 127 scales round (0.50005 scales); x' rounded to fp16 is
// another 0.062 scales off, to bf16 0.5 (half a unit of the type, of 127 scales).  Each operation rounded to fp32, one division per group.  Eight bits are what the caller asks for: they halve (fp32: quarter)
// what a layer keeps between forward and backward.  A group whose m is below 2^-120, where 127 / m leaves fp32, is kept as zeros;
// one that holds an infinity or a NaN has that as its scale and zeros as codes, so that all of it reads back as NaN.  The largest
// numbers take the largest scale whose 127-fold is finite.
//
// The gate of an expert, h = silu(a) b for rows [a | b], keeps its argument this way (hc_gated_pack) and takes from it in
// backward the gradients of a and b and h itself, which the second product's weight gradient needs (hc_gated_grad):
//   s = sigma(a');  da = dh b' s (1 + a' (1 - s));  db = dh a' s;  h' = a' s b'
// Groups do not reach over from a to b.
//
// A lane owns eight adjacent columns; group / 8 lanes share a group, whose largest magnitude goes round from lane to lane.  Bound by
// memory, one pass over each operand: 150 001 rows of 602 fp32 91 us kept (5.0 TB/s), 75 to 101 read back (4.5 to 6.0); the gate of
// 65 537 rows of 2 x 1 024 bf16 118 us forward (545 MB, 4.6 TB/s), 116 backward (680 MB, 5.9).
#include "hc_common.h"

namespace {

constexpr float PK_SMALLEST = 0x1p-120f;
constexpr float PK_LARGEST_SCALE = 0x1.0204060000000p+121f;      // 127 times the next one leaves fp32
constexpr int PK_EACH = 8;
// Eights that a lane reads before it packs the first (us, one / two / four: 150 001 rows of 608 bf16 66 / 58 / 57, of 602 fp32
// 94 / 91 / 92; 300 000 of 172 fp32 49 / 48 / 52).
constexpr int PK_AT_ONCE = 2;
// Bytes of the last-level cache.  Reading back and a pass that reads the result, plain / non-temporal stores, us: 193 MB
// 94 / 117, 361 MB 218 / 206, 722 MB 429 / 391.
constexpr int64_t PK_CACHE = 256 << 20;

// 16 bytes at the alignment of one element
typedef uint32_t pk_words_2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t pk_words_4 __attribute__((ext_vector_type(4), aligned(4)));
// N elements of S bytes at the alignment of one, as words
template <int S, int N>
struct pk_few {
  struct __attribute__((packed, aligned(S < 4 ? S : 4))) words {
    uint32_t w[S * N >= 4 ? S * N / 4 : 1];
  };
  struct __attribute__((packed, aligned(S < 4 ? S : 4))) half {
    uint16_t h;
  };
  __device__ __forceinline__ static void load(const char *p, uint32_t *w) {
    if constexpr (S * N >= 4) {
      const words q = *reinterpret_cast<const words *>(p);
#pragma unroll
      for (int i = 0; i < S * N / 4; ++i) w[i] = q.w[i];
    } else if constexpr (S * N == 2) {
      w[0] = reinterpret_cast<const half *>(p)->h;
    } else {
      w[0] = *reinterpret_cast<const uint8_t *>(p);
    }
  }
  __device__ __forceinline__ static void store(char *p, const uint32_t *w) {
    if constexpr (S * N >= 4) {
      words q;
#pragma unroll
      for (int i = 0; i < S * N / 4; ++i) q.w[i] = w[i];
      *reinterpret_cast<words *>(p) = q;
    } else if constexpr (S * N == 2) {
      reinterpret_cast<half *>(p)->h = (uint16_t)w[0];
    } else {
      *reinterpret_cast<uint8_t *>(p) = (uint8_t)w[0];
    }
  }
};

// The first 1 to 7 of eight elements of S bytes (2 S words, the others zeros): four, two and one at a time, as the bits of
// `valid` say.
template <int S>
__device__ __forceinline__ void pk_load_tail(const char *p, int valid, uint32_t (&w)[2 * S]) {
  uint32_t four[S] = {}, two[S] = {}, one[1] = {}, a[S] = {};
  if (valid & 4) pk_few<S, 4>::load(p, four);
  if (valid & 2) pk_few<S, 2>::load(p + (valid & 4) * S, two);
  if (valid & 1) pk_few<S, 1>::load(p + (valid & 6) * S, one);
  const bool pair = (valid & 2) != 0;
  if constexpr (S == 1) {
    a[0] = two[0] | one[0] << (pair ? 16 : 0);
  } else {
    a[0] = pair ? two[0] : one[0];
    if constexpr (S == 4) a[1] = two[1];
    a[S / 2] = pair ? one[0] : 0u;
  }
#pragma unroll
  for (int i = 0; i < S; ++i) {
    w[i] = valid & 4 ? four[i] : a[i];
    w[S + i] = valid & 4 ? a[i] : 0u;
  }
}

template <int S>
__device__ __forceinline__ void pk_store_tail(char *p, int valid, const uint32_t (&w)[2 * S]) {
  uint32_t a[S];
#pragma unroll
  for (int i = 0; i < S; ++i) a[i] = valid & 4 ? w[S + i] : w[i];
  if (valid & 4) pk_few<S, 4>::store(p, w);
  if (valid & 2) pk_few<S, 2>::store(p + (valid & 4) * S, a);
  const uint32_t one = valid & 2 ? (S == 1 ? a[0] >> 16 : a[S / 2]) : a[0];
  if (valid & 1) pk_few<S, 1>::store(p + (valid & 6) * S, &one);
}

// Eight adjacent elements, at no more than their own alignment; those behind `valid` read as zeros and are not written.
template <typename T>
struct pk_row {
  typedef typename std::conditional<sizeof(T) == 2, pk_words_2, pk_words_4>::type words;
  static constexpr int S = (int)sizeof(T), PIECES = S * PK_EACH / 16;
  union eight {
    words q[PIECES];
    uint32_t w[2 * S];
    T e[PK_EACH];
    __device__ eight() {}
  };
  __device__ __forceinline__ static void load(const T *__restrict__ p, int valid, float (&v)[PK_EACH]) {
    eight x;
    if (valid >= PK_EACH) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) x.q[i] = reinterpret_cast<const words *>(p)[i];
    } else if (valid > 0) {
      pk_load_tail<S>(reinterpret_cast<const char *>(p), valid, x.w);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * S; ++i) x.w[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < PK_EACH; ++i) v[i] = hc_to_f32<T>(x.e[i]);
  }
  // NT: with the non-temporal hint
  template <bool NT = false>
  __device__ __forceinline__ static void store(T *__restrict__ p, int valid, const float (&v)[PK_EACH]) {
    eight x;
#pragma unroll
    for (int i = 0; i < PK_EACH; ++i) x.e[i] = hc_from_f32<T>(v[i]);
    if (valid >= PK_EACH) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        words *at = reinterpret_cast<words *>(p) + i;
        if (NT) __builtin_nontemporal_store(x.q[i], at);
        else *at = x.q[i];
      }
    } else if (valid > 0) {
      pk_store_tail<S>(reinterpret_cast<char *>(p), valid, x.w);
    }
  }
};

struct __attribute__((packed, aligned(1))) pk_codes {
  uint32_t w[2];
};

__device__ __forceinline__ void pk_load_codes(const int8_t *__restrict__ p, int valid, float scale, float (&v)[PK_EACH]) {
  uint32_t w[2];
  if (valid >= PK_EACH) {
    const pk_codes q = *reinterpret_cast<const pk_codes *>(p);
    w[0] = q.w[0];
    w[1] = q.w[1];
  } else {
    pk_load_tail<1>(reinterpret_cast<const char *>(p), valid, w);
  }
#pragma unroll
  for (int i = 0; i < PK_EACH; ++i) v[i] = (float)(int8_t)(w[i / 4] >> (8 * (i % 4))) * scale;
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
  m = hc_join<L>(m, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
  const float most = __uint_as_float(m);
  const bool zero = most < PK_SMALLEST, bad = m >= 0x7f800000u;
  const float inverse = zero || bad ? 0.f : 1.0f / most * 127.0f;
  uint32_t w[2] = {};
#pragma unroll
  for (int i = 0; i < PK_EACH; ++i) w[i / 4] |= ((uint32_t)(int)rintf(v[i] * inverse) & 0xffu) << (8 * (i % 4));
  if (bad) w[0] = w[1] = 0;
  if (valid >= PK_EACH) {
    *reinterpret_cast<pk_codes *>(p) = pk_codes{{w[0], w[1]}};
  } else if (valid > 0) {
    pk_store_tail<1>(reinterpret_cast<char *>(p), valid, w);
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
  __device__ __forceinline__ pk_item(const PkArgs &a, uint32_t block = blockIdx.x) {
    const uint32_t t = block * HC_BLOCK + threadIdx.x, i = t / L;            // (there are less than 2^32 lanes' pieces)
    lane = (int)(t % L);
    live = i < a.items;
    const uint32_t r = live ? i / (uint32_t)a.groups : 0;
    row = r;
    g = live ? (int)(i - r * (uint32_t)a.groups) : 0;
    col = g * (L * PK_EACH) + lane * PK_EACH;
    valid = live ? a.F - col : 0;
  }
};

template <typename T, int L>
__global__ __launch_bounds__(HC_BLOCK) void pk_pack(PkArgs a, const T *__restrict__ x, int8_t *__restrict__ codes,
                                                    float *__restrict__ scale) {
  float v[PK_AT_ONCE][PK_EACH];
#pragma unroll
  for (int u = 0; u < PK_AT_ONCE; ++u) {
    const pk_item<L> it(a, blockIdx.x * PK_AT_ONCE + u);
    pk_row<T>::load(x + it.row * a.F + it.col, it.valid, v[u]);
  }
#pragma unroll
  for (int u = 0; u < PK_AT_ONCE; ++u) {
    const pk_item<L> it(a, blockIdx.x * PK_AT_ONCE + u);
    const float s = pk_encode<L>(v[u], codes + it.row * a.F + it.col, it.valid);
    if (it.live && it.lane == 0) scale[it.row * a.groups + it.g] = s;
  }
}

// NT: for a result that the last-level cache cannot hold until it is read.
template <typename T, int L, bool NT>
__global__ __launch_bounds__(HC_BLOCK) void pk_unpack(PkArgs a, const int8_t *__restrict__ codes, const float *__restrict__ scale,
                                                      T *__restrict__ x) {
  const pk_item<L> it(a);
  if (!it.live || it.valid <= 0) return;
  float v[PK_EACH];
  const int64_t at = it.row * a.F + it.col;
  pk_load_codes(codes + at, it.valid, scale[it.row * a.groups + it.g], v);
  pk_row<T>::template store<NT>(x + at, it.valid, v);
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
    pk_pack<T, decltype(lanes)::value><<<dim3((grid.x + PK_AT_ONCE - 1) / PK_AT_ONCE), dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(
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
    const auto kernel = n * F * (int64_t)sizeof(T) > PK_CACHE ? pk_unpack<T, decltype(lanes)::value, true>
                                                              : pk_unpack<T, decltype(lanes)::value, false>;
    kernel<<<grid, dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(a, codes, scale, static_cast<T *>(x));
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
