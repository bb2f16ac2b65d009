// Rows times their expert's matrix: rows offset[e] .. offset[e + 1] of x [S, K] belong to expert e with w[e] [N, K].
//
//   forward           y[s]  = x[s] w[e]^T            rows before offset[0], behind offset[E]: zeros
//   gradient of x     gx[s] = g[s] w[e]              likewise
//   gradient of w     gw[e] = sum over e's rows of g[s]^T x[s]
//
// The offsets stay on the device.  A launch has as many tiles as S rows in E groups can need at most; a block finds its expert by
// a prefix sum over the groups' tiles, and one whose number is behind the last tile ends.  The tiles are in expert_tile.h.
#include "expert_find.h"

namespace {

constexpr int EL_MAX_EXPERTS = 1024;

static bool el_sizes_ok(int64_t S, int64_t E, int64_t N, int64_t K) {
  return S < (1ll << 31) - 1 && E <= EL_MAX_EXPERTS && N <= (1 << 20) && K <= (1 << 20) && N * K < (1ll << 31);
}

static bool el_dtype_ok(int dtype) { return dtype == HC_F32 || dtype == HC_F16 || dtype == HC_BF16; }

// The result is stored in pieces of 16 bytes where its rows start on 4.
static bool el_whole(const void *out, int64_t cols, int dtype) {
  return cols * (dtype == HC_F32 ? 4 : 2) % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 4 == 0;
}

}  // namespace

extern "C" int hc_expert_linear(const void *x, int dtype, const void *w, int w_is_kn, const int64_t *offset, int64_t S,
                                int64_t E, int64_t N, int64_t K, void *out, void *stream) {
  HC_REQUIRE(S >= 0 && E >= 1 && N >= 1 && K >= 1);
  if (!el_dtype_ok(dtype)) return HC_EDTYPE;
  if (!el_sizes_ok(S, E, N, K)) return HC_EUNSUPPORTED;
  if (S == 0) return HC_OK;
  HC_REQUIRE(x && w && offset && out);
  ElProduct a = {};
  a.p = x, a.q = w, a.out = out, a.offset = offset, a.S = S;
  a.E = (int)E, a.cols = (int)N, a.inner = (int)K;
  a.whole = el_whole(out, N, dtype);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == HC_F32) return el_rows_f32(w_is_kn != 0, a, st);
  return dtype == HC_F16 ? el_rows_f16(w_is_kn != 0, a, st) : el_rows_bf16(w_is_kn != 0, a, st);
}

extern "C" size_t hc_expert_linear_grad_workspace_bytes(int64_t S, int64_t E, int64_t N, int64_t K, int dtype) {
  if (S < 0 || E < 1 || N < 1 || K < 1 || !el_dtype_ok(dtype) || !el_sizes_ok(S, E, N, K)) return 0;
  if (dtype == HC_F32) return el_grad_bytes_f32(S, E, N, K);
  return dtype == HC_F16 ? el_grad_bytes_f16(S, E, N, K) : el_grad_bytes_bf16(S, E, N, K);
}

extern "C" int hc_expert_linear_grad(const void *g, const void *x, int dtype, const int64_t *offset, int64_t S, int64_t E,
                                     int64_t N, int64_t K, void *grad_w, void *workspace, size_t workspace_bytes,
                                     void *stream) {
  HC_REQUIRE(S >= 0 && E >= 1 && N >= 1 && K >= 1);
  if (!el_dtype_ok(dtype)) return HC_EDTYPE;
  if (!el_sizes_ok(S, E, N, K)) return HC_EUNSUPPORTED;
  HC_REQUIRE(offset && grad_w && (S == 0 || (g && x)));
  ElProduct a = {};
  a.p = g, a.q = x, a.out = grad_w, a.offset = offset, a.S = S;
  a.E = (int)E, a.rows = (int)N, a.cols = (int)K;
  a.whole = el_whole(grad_w, K, dtype);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == HC_F32) return el_grad_f32(a, workspace, workspace_bytes, st);
  return dtype == HC_F16 ? el_grad_f16(a, workspace, workspace_bytes, st) : el_grad_bf16(a, workspace, workspace_bytes, st);
}
