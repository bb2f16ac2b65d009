// Rows times their expert's matrix: rows offset[e] .. offset[e + 1] of x [S, K] belong to expert e with w[e] [N, K].
//
//   forward           y[s]  = x[s] w[e]^T            rows behind offset[E]: zeros
//   gradient of x     gx[s] = g[s] w[e]              likewise
//   gradient of w     gw[e] = sum over e's rows of g[s]^T x[s]
//
// The offsets stay on the device.  A launch has as many tiles of rows as S rows in E groups can need at most; a block finds
// its expert by a prefix sum over the groups' tiles, and one whose number is behind the last tile ends.
#include "expert_find.h"

namespace {

constexpr int EL_MAX_EXPERTS = 1024;

typedef float el_acc __attribute__((ext_vector_type(4)));

struct ElArgs {
  const void *a, *w;
  void *out;
  const int64_t *offset;
  int64_t S;
  int E, N, K, tiles_n;          // out has N columns, the inner size is K
};

// Four adjacent elements, widened; those at and behind `valid` are zeros.
template <typename T>
__device__ __forceinline__ float4 el_load4(const T *p, int valid, bool whole) {
  if (valid >= 4 && whole) {
    float v[4];
    hc_vec<T, 4>::load(p, v);
    return make_float4(v[0], v[1], v[2], v[3]);
  }
  return make_float4(valid > 0 ? hc_to_f32<T>(p[0]) : 0.f, valid > 1 ? hc_to_f32<T>(p[1]) : 0.f,
                     valid > 2 ? hc_to_f32<T>(p[2]) : 0.f, valid > 3 ? hc_to_f32<T>(p[3]) : 0.f);
}

constexpr int EL_B = 64, EL_BK = 32;

// 64 rows x 64 columns of the result a block; KN: w[e] is [K, N] (the gradient of x), else [N, K].
template <typename T, bool KN>
__global__ __launch_bounds__(HC_BLOCK) void el_rows(ElArgs a, bool whole_a, bool whole_w) {
  constexpr int LDA = EL_BK + 2, LDW = KN ? EL_B + 16 : EL_BK + 2;
  __shared__ __attribute__((aligned(16))) float sa[EL_B * LDA], sw[KN ? EL_BK * LDW : EL_B * LDW];
  const int b = (int)blockIdx.x, n0 = b % a.tiles_n * EL_B;
  const ElPart tile = el_find<true>(a.offset, a.E, a.S, EL_B, b / a.tiles_n);
  if (tile.expert > a.E) return;
  const int t = (int)threadIdx.x, lane = hc_lane(), wave = hc_wave_in_block();
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32, l16 = lane & 15, g4 = lane >> 4;
  const int rows = (int)(tile.hi - tile.lo);
  const T *pa = static_cast<const T *>(a.a) + tile.lo * a.K;
  const T *pw = static_cast<const T *>(a.w) + (int64_t)(tile.expert < a.E ? tile.expert : 0) * a.N * a.K;
  T *out = static_cast<T *>(a.out) + tile.lo * a.N;
  el_acc acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = el_acc{0.f, 0.f, 0.f, 0.f};
  if (tile.expert < a.E) {
    for (int k0 = 0; k0 < a.K; k0 += EL_BK) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int f = t + i * HC_BLOCK;
        {
          const int r = f / 8, c = f % 8 * 4;
          const float4 v = el_load4(pa + (int64_t)(r < rows ? r : 0) * a.K + k0 + c, r < rows ? a.K - k0 - c : 0, whole_a);
          float *p = &sa[r * LDA + c];
          p[0] = v.x; p[1] = v.y; p[2] = v.z; p[3] = v.w;
        }
        if constexpr (KN) {
          const int r = f / 16, c = f % 16 * 4;
          const float4 v = el_load4(pw + (int64_t)(k0 + r < a.K ? k0 + r : 0) * a.N + n0 + c, k0 + r < a.K ? a.N - n0 - c : 0, whole_w);
          float *p = &sw[r * LDW + c];
          p[0] = v.x; p[1] = v.y; p[2] = v.z; p[3] = v.w;
        } else {
          const int r = f / 8, c = f % 8 * 4;
          const float4 v = el_load4(pw + (int64_t)(n0 + r < a.N ? n0 + r : 0) * a.K + k0 + c, n0 + r < a.N ? a.K - k0 - c : 0, whole_w);
          float *p = &sw[r * LDW + c];
          p[0] = v.x; p[1] = v.y; p[2] = v.z; p[3] = v.w;
        }
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < EL_BK; k += 4) {
        float x[2], y[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) x[i] = sa[(wm + i * 16 + l16) * LDA + k + g4];
#pragma unroll
        for (int j = 0; j < 2; ++j) y[j] = KN ? sw[(k + g4) * LDW + wn + j * 16 + l16] : sw[(wn + j * 16 + l16) * LDW + k + g4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[j], x[i], acc[i][j], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = wm + i * 16 + l16, c = n0 + wn + j * 16 + 4 * g4;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (r < rows && c + q < a.N) out[(int64_t)r * a.N + c + q] = hc_from_f32<T>(acc[i][j][q]);
    }
}

struct ElGradArgs {
  const void *g, *x;
  void *gw;
  const int64_t *offset;
  int64_t S;
  int E, N, K, tiles_n, tiles_k;
};

// 64 x 64 of one expert's gw a block, all of its rows.
template <typename T>
__global__ __launch_bounds__(HC_BLOCK) void el_wgrad(ElGradArgs a, bool whole_g, bool whole_x) {
  constexpr int LD = EL_B + 16;
  __shared__ __attribute__((aligned(16))) float sg[EL_BK * LD], sx[EL_BK * LD];
  const int b = (int)blockIdx.x, e = b / (a.tiles_n * a.tiles_k), in = b % (a.tiles_n * a.tiles_k);
  const int n0 = in / a.tiles_k * EL_B, c0 = in % a.tiles_k * EL_B;
  int64_t lo = a.offset[e], hi = a.offset[e + 1];
  lo = lo < 0 ? 0 : lo > a.S ? a.S : lo;
  hi = hi < lo ? lo : hi > a.S ? a.S : hi;
  const int t = (int)threadIdx.x, lane = hc_lane(), wave = hc_wave_in_block();
  const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32, l16 = lane & 15, g4 = lane >> 4;
  const T *g = static_cast<const T *>(a.g), *x = static_cast<const T *>(a.x);
  el_acc acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = el_acc{0.f, 0.f, 0.f, 0.f};
  for (int64_t s0 = lo; s0 < hi; s0 += EL_BK) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int f = t + i * HC_BLOCK, r = f / 16, c = f % 16 * 4;
      const bool in_rows = s0 + r < hi;
      const int64_t s = in_rows ? s0 + r : lo;
      const float4 u = el_load4(g + s * a.N + n0 + c, in_rows ? a.N - n0 - c : 0, whole_g);
      const float4 v = el_load4(x + s * a.K + c0 + c, in_rows ? a.K - c0 - c : 0, whole_x);
      float *p = &sg[r * LD + c], *q = &sx[r * LD + c];
      p[0] = u.x; p[1] = u.y; p[2] = u.z; p[3] = u.w;
      q[0] = v.x; q[1] = v.y; q[2] = v.z; q[3] = v.w;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EL_BK; k += 4) {
      float u[2], v[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        u[i] = sg[(k + g4) * LD + wm + i * 16 + l16];
        v[i] = sx[(k + g4) * LD + wn + i * 16 + l16];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j], u[i], acc[i][j], 0, 0, 0);
    }
  }
  T *gw = static_cast<T *>(a.gw) + (int64_t)e * a.N * a.K;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = n0 + wm + i * 16 + l16, c = c0 + wn + j * 16 + 4 * g4;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (r < a.N && c + q < a.K) gw[(int64_t)r * a.K + c + q] = hc_from_f32<T>(acc[i][j][q]);
    }
}

template <typename F>
static int el_with_type(int dtype, F &&f) {
  if (dtype == HC_F32) return f(float{});
  return HC_EDTYPE;
}

static bool el_sizes_ok(int64_t S, int64_t E, int64_t N, int64_t K) {
  return S < (1ll << 31) - 1 && E <= EL_MAX_EXPERTS && N <= (1 << 20) && K <= (1 << 20) && N * K < (1ll << 31);
}

template <typename T>
static bool el_whole(const void *p, int64_t width) {
  return width % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0;
}

}  // namespace

extern "C" int hc_expert_linear(const void *x, int dtype, const void *w, int w_is_kn, const int64_t *offset, int64_t S,
                                int64_t E, int64_t N, int64_t K, void *out, void *stream) {
  HC_REQUIRE(S >= 0 && E >= 1 && N >= 1 && K >= 1);
  if (!el_sizes_ok(S, E, N, K)) return HC_EUNSUPPORTED;
  if (S == 0) return dtype >= HC_F32 && dtype <= HC_BF16 ? HC_OK : HC_EDTYPE;
  HC_REQUIRE(x && w && offset && out);
  if (dtype == HC_F16 || dtype == HC_BF16) {
    ElProduct p = {};
    p.p = x, p.q = w, p.out = out, p.offset = offset, p.S = S;
    p.E = (int)E, p.cols = (int)N, p.inner = (int)K;
    return el_half_rows(dtype, w_is_kn != 0, p, static_cast<hipStream_t>(stream));
  }
  return el_with_type(dtype, [&](auto type) {
    typedef decltype(type) T;
    ElArgs a = {x, w, out, offset, S, (int)E, (int)N, (int)K, (int)((N + EL_B - 1) / EL_B)};
    const int64_t blocks = (S / EL_B + E + 1) * a.tiles_n;
    if (!hc_grid_ok(blocks)) return (int)HC_EUNSUPPORTED;
    const auto kernel = w_is_kn ? el_rows<T, true> : el_rows<T, false>;
    kernel<<<dim3((unsigned)blocks), dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(
        a, el_whole<T>(x, K), el_whole<T>(w, w_is_kn ? N : K));
    return hc_launch_status();
  });
}

extern "C" size_t hc_expert_linear_grad_workspace_bytes(int64_t S, int64_t E, int64_t N, int64_t K, int dtype) {
  if (S < 0 || E < 1 || N < 1 || K < 1 || !el_sizes_ok(S, E, N, K)) return 0;
  return dtype == HC_F32 ? 0 : el_half_grad_bytes(S, E, N, K);
}

extern "C" int hc_expert_linear_grad(const void *g, const void *x, int dtype, const int64_t *offset, int64_t S, int64_t E,
                                     int64_t N, int64_t K, void *grad_w, void *workspace, size_t workspace_bytes,
                                     void *stream) {
  HC_REQUIRE(S >= 0 && E >= 1 && N >= 1 && K >= 1);
  if (!el_sizes_ok(S, E, N, K)) return HC_EUNSUPPORTED;
  HC_REQUIRE(offset && grad_w && (S == 0 || (g && x)));
  if (dtype == HC_F16 || dtype == HC_BF16) {
    ElProduct p = {};
    p.p = g, p.q = x, p.out = grad_w, p.offset = offset, p.S = S;
    p.E = (int)E, p.rows = (int)N, p.cols = (int)K;
    return el_half_grad(dtype, p, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
  }
  return el_with_type(dtype, [&](auto type) {
    typedef decltype(type) T;
    ElGradArgs a = {g, x, grad_w, offset, S, (int)E, (int)N, (int)K, (int)((N + EL_B - 1) / EL_B), (int)((K + EL_B - 1) / EL_B)};
    const int64_t blocks = E * a.tiles_n * a.tiles_k;
    if (!hc_grid_ok(blocks)) return (int)HC_EUNSUPPORTED;
    el_wgrad<T><<<dim3((unsigned)blocks), dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(a, el_whole<T>(g, N),
                                                                                                el_whole<T>(x, K));
    return hc_launch_status();
  });
}
