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
// memory, one pass over each operand: 150 001 rows of 602 fp32 81 us kept (5.6 TB/s), 75 to 101 read back (4.5 to 6.0); the gate of
// 65 537 rows of 2 x 1 024 bf16 118 us forward (545 MB, 4.6 TB/s), 116 backward (680 MB, 5.9).
#include "packed_rows.h"

namespace {

// Eights that a lane reads before it packs the first (us, one / two / four: 150 001 rows of 608 bf16 66 / 58 / 57, of 602 fp32
// 94 / 91 / 92; 300 000 of 172 fp32 49 / 48 / 52).
constexpr int PK_AT_ONCE = 2;
// Bytes of the last-level cache.  Reading back and a pass that reads the result, plain / non-temporal stores, us: 193 MB
// 94 / 117, 361 MB 218 / 206, 722 MB 429 / 391.
constexpr int64_t PK_CACHE = 256 << 20;

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
