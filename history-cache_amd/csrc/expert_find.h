// Which rows a block of an expert product works on, found from the offsets in device memory.
#pragma once

#include "hc_common.h"

// Part `part` of the `parts` that expert `expert`'s rows are cut into.  Every wave of a block looks for it and finds the same.
struct ElPart {
  int expert;            // E, E + 1: the rows behind the last expert, before the first; E + 2: there is no such part
  int part, parts;
  int place;             // parts before it, counting experts of several parts only (where its partial sums lie)
  int64_t lo, hi;        // its rows
};

__device__ __forceinline__ int el_scan(int v) {
  const int lane = hc_lane();
#pragma unroll
  for (int d = 1; d < HC_WAVE; d *= 2) {
    const int o = __shfl_up(v, d, HC_WAVE);
    if (lane >= d) v += o;
  }
  return v;
}

// Rows offset[e] .. offset[e + 1] of the lane's expert e, for e = E the rows behind the last expert, none for a larger one.  An offset outside [0, S] counts as the end that it lies behind, one below an earlier one as that one: whatever the offsets
// are, no two experts have a row in common.  most: the largest offset of the experts before the first lane's, then of all.
__device__ __forceinline__ void el_rows_of(const int64_t *__restrict__ offset, int E, int64_t S, int e, int *most, int64_t *lo,
                                           int64_t *hi) {
  const auto inside = [&](int64_t a) { return (int)(a < 0 ? 0 : a > S ? S : a); };        // (S is below 2^31)
  int a = e <= E ? inside(offset[e]) : (int)S;
  const int b = e < E ? inside(offset[e + 1]) : (int)S;
  if (__ballot(b < a) != 0 || __builtin_amdgcn_readfirstlane(a) < *most) {
    const int lane = hc_lane();
    a = a > *most ? a : *most;
#pragma unroll
    for (int d = 1; d < HC_WAVE; d *= 2) {
      const int o = __shfl_up(a, d, HC_WAVE);
      if (lane >= d && o > a) a = o;
    }
  }
  *lo = a;
  *hi = a > b ? a : b;
  *most = __builtin_amdgcn_readlane(a > b ? a : b, HC_WAVE - 1);
}

// The t-th piece of up to `rows` rows, expert by expert; the rows behind the last expert follow as expert E, those before the
// first as E + 1.
__device__ __forceinline__ ElPart el_find_rows(const int64_t *__restrict__ offset, int E, int64_t S, int rows, int t) {
  const int lane = hc_lane();
  int before = 0, most = 0;
  for (int e0 = 0; e0 <= E + 1; e0 += HC_WAVE) {
    int64_t lo, hi;
    el_rows_of(offset, E, S, e0 + lane, &most, &lo, &hi);
    if (e0 + lane == E + 1) {
      const int64_t first = offset[0];
      lo = 0;
      hi = first < 0 ? 0 : first > S ? S : first;
    }
    const int parts = (int)((hi - lo + rows - 1) / rows), upto = el_scan(parts);
    const uint64_t in = __ballot(t < before + upto);
    if (in != 0) {
      const int l = __ffsll((long long)in) - 1;
      ElPart r = {};
      r.expert = e0 + l;
      r.parts = __builtin_amdgcn_readlane(parts, l);
      r.part = t - (before + __builtin_amdgcn_readlane(upto, l) - r.parts);
      r.lo = hc_readlane64(lo, l) + (int64_t)r.part * rows;
      const int64_t end = hc_readlane64(hi, l);
      r.hi = r.lo + rows < end ? r.lo + rows : end;
      return r;
    }
    before += __builtin_amdgcn_readlane(upto, HC_WAVE - 1);
  }
  ElPart r = {};
  r.expert = E + 2;
  return r;
}

// The t-th part of up to `rows` rows for the experts' gradients; an expert without rows has one of none (its gradient is zeros).
// The parts of `rows` rows come first, then the experts' last, shorter ones, of up to 64 experts the longest first: what is
// started last is short.  The order changes no result.
__device__ __forceinline__ ElPart el_find_part(const int64_t *__restrict__ offset, int E, int64_t S, int64_t rows, int t) {
  const int lane = hc_lane();
  for (int last = 0; last < 2; ++last) {
    int before = 0, several = 0, most = 0;
    for (int e0 = 0; e0 < E; e0 += HC_WAVE) {
      int64_t lo, hi;
      el_rows_of(offset, E, S, e0 + lane < E ? e0 + lane : E + 1, &most, &lo, &hi);
      const int full = (int)((hi - lo) / rows), rest = (int)(hi - lo - full * rows);
      const bool short_one = e0 + lane < E && (rest > 0 || full == 0);
      const int parts = full + (short_one ? 1 : 0), many = parts > 1 ? parts : 0, place = several + el_scan(many) - many;
      const int mine = last ? (short_one ? 1 : 0) : full, upto = before + el_scan(mine);
      uint64_t in;
      if (last && E <= HC_WAVE) {
        int rank = 0;
        for (int l = 0; l < E; ++l) {
          const int other = __builtin_amdgcn_readlane(short_one ? rest : -1, l);
          rank += other > rest || (other == rest && l < lane) ? 1 : 0;
        }
        in = __ballot(short_one && rank == t);
      } else {
        in = __ballot(t < upto);
      }
      if (in != 0) {
        const int l = __ffsll((long long)in) - 1;
        ElPart r;
        r.expert = e0 + l;
        r.parts = __builtin_amdgcn_readlane(parts, l);
        r.part = last ? __builtin_amdgcn_readlane(full, l) : t - __builtin_amdgcn_readlane(upto - mine, l);
        r.place = __builtin_amdgcn_readlane(place, l) + r.part;
        r.lo = hc_readlane64(lo, l) + r.part * rows;
        const int64_t end = hc_readlane64(hi, l);
        r.hi = r.lo + rows < end ? r.lo + rows : end;
        return r;
      }
      before = __builtin_amdgcn_readlane(upto, HC_WAVE - 1);
      several = __builtin_amdgcn_readlane(place + many, HC_WAVE - 1);
    }
    t -= before;
  }
  ElPart r = {};
  r.expert = E + 2;
  return r;
}

// A product for the kernels of expert_tile.h.
struct ElProduct {
  const void *p, *q;            // rows of the result come from p, columns from q
  void *out;
  const int64_t *offset;
  int64_t S;
  int E, rows, cols, inner;     // rows: of one expert's gradient (by rows of the batch: unused)
  int tiles_p, tiles_q;
  int64_t slab;                 // rows of the batch in one part of a gradient
  float *part;                  // their partial sums
  bool whole;                   // the result is stored in pieces of 16 bytes
};

// expert_f32.hip, expert_f16.hip, expert_bf16.hip (arguments are checked by the callers).
#define EL_DECLARE(name)                                                                                              \
  __attribute__((visibility("hidden"))) int el_rows_##name(bool w_is_kn, const ElProduct &a, hipStream_t st);        \
  __attribute__((visibility("hidden"))) size_t el_grad_bytes_##name(int64_t S, int64_t E, int64_t N, int64_t K);     \
  __attribute__((visibility("hidden"))) int el_grad_##name(const ElProduct &a, void *workspace, size_t workspace_bytes, hipStream_t st)
EL_DECLARE(f32);
EL_DECLARE(f16);
EL_DECLARE(bf16);
