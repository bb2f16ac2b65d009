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
// Forward: a wave takes 64 / L rows.  It reads them whole, puts into LDS what is compared (c, or l without a bias) as fp32, and each
// row is then gone through by L lanes, every one with the K + 1 largest of its share in registers, sorted: a 64-bit number whose
// upper half is c and whose lower half falls with the index orders, read as fp64, by both, so that a new one moves through the list
// with one maximum and one minimum a place.  The lists of a row's lanes are put together at the end.  c in fp32 is off by up to 2^-21 or so:
// where neighbours among the first K + 1, or the last open and the first closed group, are nearer than that and do not come from equal
// numbers, the wave decides the row again in fp64, all lanes on it.
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
  int dtype, E, k, groups, per_group, top_group;
  int quads, stride, rank_stride;      // in LDS: pieces of four a row, floats from one row to the next, and from one row's ranks
  bool softmax, normalize, whole;
};

__device__ __forceinline__ int64_t rs_bits(double v) { return __builtin_bit_cast(int64_t, v); }
__device__ __forceinline__ double rs_double(int64_t v) { return __builtin_bit_cast(double, v); }
__device__ __forceinline__ float rs_closed() { return -__builtin_inff(); }

// ---- the exact way: one row by a whole wave
// fp64 as whole numbers that order like it: NaN above everything, CLOSED below.
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
__device__ __forceinline__ int64_t rs_shfl(int64_t v, int lane) {
  const int lo = __shfl((int)(uint32_t)(uint64_t)v, lane, HC_WAVE), hi = __shfl((int)((uint64_t)v >> 32), lane, HC_WAVE);
  return (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
}

template <typename T>
__device__ __forceinline__ float rs_logit(const RsArgs &a, int64_t at) {
  return hc_to_f32<T>(static_cast<const T *>(a.logits)[at]);
}
__device__ __forceinline__ float rs_logit(const RsArgs &a, int64_t at) {
  if (a.dtype == HC_F32) return rs_logit<float>(a, at);
  if (a.dtype == HC_F16) return rs_logit<__half>(a, at);
  return rs_logit<__hip_bfloat16>(a, at);
}

// The winners of row r into won[0 .. k) (-1: none).  key: E numbers in LDS.
__device__ __forceinline__ void rs_choose_exactly(const RsArgs &a, int64_t r, int64_t *key, int *won) {
  const int lane = hc_lane();
  const auto larger = [](int64_t x, int64_t y) { return x > y ? x : y; };
  double top = -__builtin_inf(), sum = 0.0;
  if (a.softmax) {
    for (int e = lane; e < a.E; e += HC_WAVE) {
      const float l = rs_logit(a, r * a.E + e);
      top = l > top ? (double)l : top;
    }
    top = rs_value(hc_join<HC_WAVE>(rs_order(top), larger));
    for (int e = lane; e < a.E; e += HC_WAVE) {
      const float l = rs_logit(a, r * a.E + e);
      sum += rt_masked(l) ? 0.0 : exp((double)l - top);
    }
    sum = rs_double(hc_join<HC_WAVE>(rs_bits(sum), [](int64_t x, int64_t y) { return rs_bits(rs_double(x) + rs_double(y)); }));
  }
  const auto score = [&](float l) {
    return rt_masked(l) ? 0.0 : a.softmax ? exp((double)l - top) / sum : 1.0 / (1.0 + exp(-(double)l));
  };
  for (int e = lane; e < a.E; e += HC_WAVE) {
    const float l = rs_logit(a, r * a.E + e);
    key[e] = rt_masked(l) ? RS_CLOSED : rs_order(score(l) + (a.bias != nullptr ? (double)a.bias[e] : 0.0));
  }
  rt_in_order();
  uint64_t open = ~0ull;
  if (a.groups > 1) {
    int64_t first = RS_CLOSED, second = RS_CLOSED;
    if (lane < a.groups)
      for (int j = 0; j < a.per_group; ++j) {
        const int64_t c = key[lane * a.per_group + j];
        second = c > first ? first : c > second ? c : second;
        first = c > first ? c : first;
      }
    const int64_t rank = second == RS_CLOSED ? first : rs_order(rs_value(first) + rs_value(second));
    int ahead = 0;
    for (int h = 0; h < a.groups; ++h) {
      const int64_t other = rs_shfl(rank, h);
      if (other > rank || (other == rank && h < lane)) ++ahead;
    }
    open = __ballot(lane < a.groups && ahead < a.top_group);
    rt_in_order();
  }
  // (without a bias experts are compared by their logits)
  for (int e = lane; e < a.E; e += HC_WAVE) {
    if (a.groups > 1 && (open >> (e / a.per_group) & 1) == 0) key[e] = RS_CLOSED;
    else if (a.bias == nullptr && key[e] != RS_CLOSED) key[e] = rs_order((double)rs_logit(a, r * a.E + e));
  }
  rt_in_order();
  for (int j = 0; j < a.k; ++j) {
    int64_t best = RS_CLOSED;
    uint32_t at = 0xffffffffu;
    for (int e = lane; e < a.E; e += HC_WAVE)
      if (key[e] > best) best = key[e], at = (uint32_t)e;
    const int64_t most = hc_join<HC_WAVE>(best, larger);
    const uint32_t e = hc_join<HC_WAVE>(best == most ? at : 0xffffffffu, [](uint32_t x, uint32_t y) { return x < y ? x : y; });
    rt_in_order();
    if (e != 0xffffffffu && (int)(e % HC_WAVE) == lane) key[e] = RS_CLOSED;
    if (lane == 0) won[j] = (int)e;
    rt_in_order();
  }
}

// ---- the fast way
// c and the index of an expert as one number: larger c first, of equal ones the lower index.
__device__ __forceinline__ double rs_key(float c, int e) {
  const uint32_t hi = __float_as_uint(c), lo = (uint32_t)((int32_t)hi >> 31) ^ ~(uint32_t)e;
  return rs_double((int64_t)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ float rs_key_value(double k) { return __uint_as_float((uint32_t)((uint64_t)rs_bits(k) >> 32)); }
__device__ __forceinline__ int rs_key_index(double k) {
  const uint64_t b = (uint64_t)rs_bits(k);
  return (int)~((uint32_t)b ^ (uint32_t)((int64_t)b >> 63));
}

__device__ __forceinline__ void rs_in_order(double &x, double &y) {
  const double low = __builtin_fmin(x, y);
  x = __builtin_fmax(x, y);
  y = low;
}

// The N largest numbers so far, sorted, and the largest of the others.
template <int N>
struct rs_list {
  double t[N], out;
  __device__ __forceinline__ rs_list() {
#pragma unroll
    for (int j = 0; j < N; ++j) t[j] = rs_key(rs_closed(), 0);
    out = t[0];
  }
  // M sorted numbers more: the last M here meet them the other way round, which leaves the N largest of all in two runs.
  template <int M>
  __device__ __forceinline__ void take(const double (&o)[M]) {
#pragma unroll
    for (int j = 0; j < M; ++j) {
      const double mine = t[N - M + j], other = o[M - 1 - j];
      t[N - M + j] = __builtin_fmax(mine, other);
      out = __builtin_fmax(out, __builtin_fmin(mine, other));
    }
#pragma unroll
    for (int d = N / 2; d >= 1; d /= 2)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if ((i & d) == 0) rs_in_order(t[i], t[i + d]);
  }
  __device__ __forceinline__ void take_four(float4 v, int e) {
    double o[4] = {rs_key(v.x, e), rs_key(v.y, e + 1), rs_key(v.z, e + 2), rs_key(v.w, e + 3)};
    rs_in_order(o[0], o[1]);
    rs_in_order(o[2], o[3]);
    rs_in_order(o[0], o[2]);
    rs_in_order(o[1], o[3]);
    rs_in_order(o[1], o[2]);
    if constexpr (N >= 4) {
      take(o);
    } else {
      const double two[2] = {o[0], o[1]};
      out = __builtin_fmax(out, o[2]);
      take(two);
    }
  }
  // The list of the row that L lanes have, in each of them.
  template <int L, int D = 1>
  __device__ __forceinline__ void join() {
    if constexpr (D < L) {
      double o[N];
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] = rs_double(hc_other<D>(rs_bits(t[j])));
      out = __builtin_fmax(out, rs_double(hc_other<D>(rs_bits(out))));
      take(o);
      join<L, 2 * D>();
    }
  }
};

// 1 / (1 + exp(-l)) by the instructions, within 2^-22.
__device__ __forceinline__ float rs_near_sigma(float l) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(l * -1.44269504f));
}
__device__ __forceinline__ float rs_sigma(float l) {
  const float e = expf(-fabsf(l));
  return (l < 0.f ? e : 1.f) / (1.f + e);
}

// What is compared, as it lies in LDS: no -0, one NaN (another could make no number of a key).
__device__ __forceinline__ float rs_plain(float c) { return c != c ? __uint_as_float(0x7fc00000u) : c + 0.f; }
// c of a logit and a bias that is plain: s is not below 0.
__device__ __forceinline__ float rs_choice(float l, float bias) {
  const int32_t c = __builtin_bit_cast(int32_t, fabsf(rs_near_sigma(l)) + bias);
  return rt_masked(l) ? rs_closed() : __builtin_bit_cast(float, c < 0x7fc00000 ? c : 0x7fc00000);
}

// Rows r0 .. r0 + rows into LDS: c where the score is a logit's own and there is a bias, l otherwise.
template <typename T>
__device__ __forceinline__ void rs_stage(const RsArgs &a, int64_t r0, int rows, float *s, const float *bias) {
  constexpr int PIECE = 16 / (int)sizeof(T), AT_ONCE = 4;
  const int lane = hc_lane();
  const T *from = static_cast<const T *>(a.logits) + r0 * a.E;
  const bool make = a.bias != nullptr && !a.softmax;
  if (a.whole) {
    const int pieces = rows * (a.E / PIECE), each = a.E / PIECE, down = HC_WAVE / each, across = HC_WAVE % each;
    int row = lane / each, col = lane % each;
    for (int q0 = lane; q0 < pieces; q0 += AT_ONCE * HC_WAVE) {
      typename hc_vec<T, PIECE>::U u[AT_ONCE];
#pragma unroll
      for (int t = 0; t < AT_ONCE; ++t) {
        const int q = q0 + t * HC_WAVE;
        u[t].raw = *reinterpret_cast<const typename hc_vec<T, PIECE>::raw_t *>(from + (q < pieces ? q : q0) * PIECE);
      }
#pragma unroll
      for (int t = 0; t < AT_ONCE; ++t) {
        if (q0 + t * HC_WAVE < pieces) {
          float v[PIECE];
#pragma unroll
          for (int i = 0; i < PIECE; ++i) v[i] = hc_to_f32<T>(u[t].e[i]);
#pragma unroll
          for (int i = 0; i < PIECE; i += 4) {
            if (make) {
              const float4 b = *reinterpret_cast<const float4 *>(bias + col * PIECE + i);
              v[i] = rs_choice(v[i], b.x);
              v[i + 1] = rs_choice(v[i + 1], b.y);
              v[i + 2] = rs_choice(v[i + 2], b.z);
              v[i + 3] = rs_choice(v[i + 3], b.w);
            } else {
#pragma unroll
              for (int j = 0; j < 4; ++j) v[i + j] = rs_plain(v[i + j]);
            }
            *reinterpret_cast<float4 *>(s + row * a.stride + col * PIECE + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          }
        }
        row += down;
        col += across;
        if (col >= each) col -= each, ++row;
      }
    }
  } else {
    const int all = rows * a.E, down = HC_WAVE / a.E, across = HC_WAVE % a.E;
    int row = lane / a.E, col = lane % a.E;
    for (int x = lane; x < all; x += HC_WAVE) {
      const float v = hc_to_f32<T>(from[x]);
      s[row * a.stride + col] = make ? rs_choice(v, bias[col]) : rs_plain(v);
      row += down;
      col += across;
      if (col >= a.E) col -= a.E, ++row;
    }
    for (int x = lane; x < rows * 4; x += HC_WAVE)            // the rest of a row's last four
      if (a.E + x % 4 < 4 * a.quads) s[x / 4 * a.stride + a.E + x % 4] = rs_closed();
  }
}

// Calls f(four values, index of the first) for the elements from .. to of a row in LDS that lane `sub` of L takes; behind `to`: closed.
template <int L, typename F>
__device__ __forceinline__ void rs_each(const float *row, int from, int to, int sub, bool by_four, F &&f) {
  if (by_four) {
    for (int e = from + 4 * sub; e < to; e += 4 * L) f(*reinterpret_cast<const float4 *>(row + e), e);
  } else {
    for (int e = from + 4 * sub; e < to; e += 4 * L)
      f(make_float4(row[e], e + 1 < to ? row[e + 1] : rs_closed(), e + 2 < to ? row[e + 2] : rs_closed(),
                    e + 3 < to ? row[e + 3] : rs_closed()), e);
  }
}

template <int L, typename F>
__device__ __forceinline__ double rs_join(double v, F &&f) {
  return rs_double(hc_join<L>(rs_bits(v), [&](int64_t x, int64_t y) { return rs_bits(f(rs_double(x), rs_double(y))); }));
}

// K: places for winners, k <= K; L: lanes a row.
template <int K, int L>
__global__ __launch_bounds__(HC_WAVE) void rs_forward(RsArgs a) {
  // rows, the groups' ranks of each, the bias
  extern __shared__ __attribute__((aligned(16))) float s_all[];
  constexpr int ROWS = HC_WAVE / L;
  const int lane = hc_lane(), sub = lane % L, mine = lane / L;
  const int64_t r0 = (int64_t)blockIdx.x * ROWS;
  const int rows = a.n - r0 < ROWS ? (int)(a.n - r0) : ROWS;
  const bool live = mine < rows;
  const int64_t r = r0 + (live ? mine : 0);
  float *bias = s_all + ROWS * (a.stride + a.rank_stride);
  if (a.bias != nullptr) {
    for (int e = lane; e < a.E; e += HC_WAVE) bias[e] = rs_plain(a.bias[e]);
    rt_in_order();
  }
  if (a.dtype == HC_F32) rs_stage<float>(a, r0, rows, s_all, bias);
  else if (a.dtype == HC_F16) rs_stage<__half>(a, r0, rows, s_all, bias);
  else rs_stage<__hip_bfloat16>(a, r0, rows, s_all, bias);
  rt_in_order();
  float *row = s_all + (live ? mine : 0) * a.stride;
  float top = rs_closed(), all = 0.f;
  if (a.softmax) {
    rs_each<L>(row, 0, 4 * a.quads, sub, true, [&](float4 l, int) { top = fmaxf(top, fmaxf(fmaxf(l.x, l.y), fmaxf(l.z, l.w))); });
    top = hc_join<L>(top, [](float x, float y) { return fmaxf(x, y); });
    double sum = 0.0;
    const auto e = [&](float l) { return rt_masked(l) ? 0.f : expf(l - top); };
    rs_each<L>(row, 0, 4 * a.quads, sub, true, [&](float4 l, int) {
      sum += ((double)e(l.x) + (double)e(l.y)) + ((double)e(l.z) + (double)e(l.w));
    });
    sum = rs_join<L>(sum, [](double x, double y) { return x + y; });
    all = (float)sum;
    if (a.bias != nullptr) {
      rt_in_order();
      if (live)
        for (int e = sub; e < a.E; e += L) {
          const float l = row[e];
          row[e] = rt_masked(l) ? l : rs_plain(expf(l - top) / all + bias[e]);
        }
      rt_in_order();
    }
  }
  const bool exact = a.bias == nullptr;              // what is compared are logits
  bool near = false;                                 // too near for fp32
  uint64_t open = ~0ull;
  const bool by_four = a.per_group % 4 == 0;
  if (a.groups > 1) {
    float *rank = s_all + ROWS * a.stride + mine * a.rank_stride;
    for (int g = 0; g < a.groups; ++g) {
      float first = rs_closed(), second = rs_closed();
      // (a NaN makes the sum one, whose group is decided again)
      float nan = 0.f;
      const auto more = [&](float c) {
        second = fmaxf(second, fminf(first, c));
        first = fmaxf(first, c);
      };
      rs_each<L>(row, g * a.per_group, (g + 1) * a.per_group, sub, by_four, [&](float4 c, int) {
        const float x = fmaxf(c.x, c.y), y = fminf(c.x, c.y), z = fmaxf(c.z, c.w), w = fminf(c.z, c.w);
        second = fmaxf(fmaxf(second, fmaxf(y, w)), fminf(fmaxf(x, z), fmaxf(first, fminf(x, z))));
        first = fmaxf(first, fmaxf(x, z));
        nan = c.x != c.x || c.y != c.y || c.z != c.z || c.w != c.w ? __builtin_nanf("") : nan;
      });
#pragma unroll
      for (int d = 1; d < L; d *= 2) {
        const float f = __shfl_xor(first, d, HC_WAVE), s = __shfl_xor(second, d, HC_WAVE);
        nan += __shfl_xor(nan, d, HC_WAVE);
        second = fmaxf(second, s);
        more(f);
      }
      near = near || nan != nan;
      if (exact && !rt_masked(first)) {
        first = a.softmax ? expf(first - top) : rs_sigma(first);
        second = a.softmax ? expf(second - top) : rs_sigma(second);
      }
      if (sub == 0) rank[g] = rt_masked(first) ? first : rt_masked(second) ? first : first + second;
    }
    rt_in_order();
    // the last open group and the first closed one
    float least = -rs_closed(), most = rs_closed();
    open = 0;
    for (int g = sub; g < a.groups; g += L) {
      const float own = rank[g];
      int ahead = 0;
      for (int h = 0; h < a.groups; ++h) {
        const float other = rank[h];
        ahead += other > own || (other == own && h < g) ? 1 : 0;
      }
      if (ahead < a.top_group) open |= 1ull << g, least = fminf(least, own);
      else most = fmaxf(most, own);
    }
    open = (uint64_t)hc_join<L>((int64_t)open, [](int64_t x, int64_t y) { return x | y; });
    least = hc_join<L>(least, [](float x, float y) { return fminf(x, y); });
    most = hc_join<L>(most, [](float x, float y) { return fmaxf(x, y); });
    const float off = exact ? 0x1p-16f * fabsf(least) : 0x1p-19f * (1.f + fabsf(least));
    near = near || (!rt_masked(most) && !(least - most > off));
  }
  rs_list<K> list;
  if (a.groups > 1) {
    uint64_t left = open;
    for (int t = 0; t < a.top_group; ++t) {
      const int g = left != 0 ? __builtin_ctzll(left) : 0;
      left &= left - 1;
      rs_each<L>(row, g * a.per_group, (g + 1) * a.per_group, sub, by_four, [&](float4 c, int e) { list.take_four(c, e); });
    }
  } else {
    rs_each<L>(row, 0, 4 * a.quads, sub, true, [&](float4 c, int e) { list.take_four(c, e); });
  }
  list.template join<L>();
  int won[K];
  float p[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    won[j] = j < a.k && !rt_masked(rs_key_value(list.t[j])) ? rs_key_index(list.t[j]) : -1;
    p[j] = won[j] >= 0 ? rs_logit(a, r * a.E + won[j]) : 0.f;
  }
  if (!exact) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const double next = j + 1 < K ? list.t[j + 1] : list.out;
      const float c = rs_key_value(list.t[j]), d = rs_key_value(next);
      if (j < a.k && !rt_masked(d) && !(c - d > 0x1p-20f * (1.f + fabsf(c)))) {
        const int y = rs_key_index(next);
        // (equal numbers: the lower index is the right one)
        if (!(p[j] == rs_logit(a, r * a.E + y) && bias[won[j]] == bias[y])) near = true;
      }
    }
  }
  uint64_t again = __ballot(near && live && sub == 0);
  if (again != 0) {
    int64_t *key = reinterpret_cast<int64_t *>(s_all);
    int *found = reinterpret_cast<int *>(key + a.E);
    rt_in_order();
    while (again != 0) {
      const int row_of = __builtin_ctzll(again) / L;
      again &= again - 1;
      rs_choose_exactly(a, r0 + row_of, key, found);
      if (mine == row_of) {
#pragma unroll
        for (int j = 0; j < K; ++j) {
          won[j] = j < a.k ? found[j] : -1;
          p[j] = won[j] >= 0 ? rs_logit(a, r * a.E + won[j]) : 0.f;
        }
      }
      rt_in_order();
    }
  }
  float s[K], sum = 0.f;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    s[j] = won[j] < 0 ? 0.f : a.softmax ? expf(p[j] - top) : rs_sigma(p[j]);
    sum += s[j];
  }
  const float of = a.normalize ? (all != all ? all : sum) : a.softmax ? all : 1.f;
  if (!live) return;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    if (j >= a.k || j % L != sub) continue;
    a.expert[r * a.k + j] = won[j];
    a.weight[r * a.k + j] = won[j] < 0 || of == 0.f ? 0.f : a.scale * (s[j] / of);
    if (a.picked != nullptr) a.picked[r * a.k + j] = p[j];
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
  if (dtype < HC_F32 || dtype > HC_BF16) return HC_EDTYPE;
  RsArgs a{logits, bias, expert, weight, picked, n, scale, dtype, (int)E, (int)top_k,
           // (all groups open: as if there were one)
           top_group == num_group ? 1 : (int)num_group, (int)(E / num_group), (int)top_group, 0, 0, 0, score != RS_SIGMOID,
           normalize != 0, false};
  a.whole = dtype == HC_F32 ? rt_row<float, 4>::whole(logits, E) : rt_row<__half, 8>::whole(logits, E);
  a.quads = (int)((E + 3) / 4);
  const auto launch = [&](auto places, auto lanes) {
    constexpr int L = decltype(lanes)::value;
    const int64_t blocks = (n + HC_WAVE / L - 1) / (HC_WAVE / L);
    if (!hc_grid_ok(blocks)) return (int)HC_EUNSUPPORTED;
    // rows lie so that lanes which read side by side read from other banks
    int from_row = a.quads;
    while (L < 8 && from_row % 8 != L) ++from_row;
    a.stride = 4 * from_row;
    a.rank_stride = a.groups > 1 ? a.groups | 1 : 0;
    if (HC_WAVE / L < 4) a.rank_stride = (a.rank_stride + 3) / 4 * 4;         // (what follows lies at a multiple of 16 bytes)
    const size_t rows = ((size_t)(HC_WAVE / L) * (a.stride + a.rank_stride) + (bias ? (size_t)E : 0)) * sizeof(float);
    const size_t exactly = (size_t)E * sizeof(int64_t) + RT_MAX_CHOICES * sizeof(int);
    rs_forward<decltype(places)::value, L><<<dim3((unsigned)blocks), dim3(HC_WAVE), rows > exactly ? rows : exactly,
                                             static_cast<hipStream_t>(stream)>>>(a);
    return hc_launch_status();
  };
  const auto with_lanes = [&](auto places) {
    // as few lanes a row as keep its wave's rows under 18 KB of LDS (nine waves a compute unit), more where rows are few
    const int least = E <= 64 ? 1 : E <= 256 ? 4 : 16;
    int lanes = least;
    while (lanes < 64 && lanes < a.quads && n * lanes < 64 * 2048) lanes *= 4;
    if (lanes == 1) return launch(places, std::integral_constant<int, 1>{});
    if (lanes == 4) return launch(places, std::integral_constant<int, 4>{});
    if (lanes == 16) return launch(places, std::integral_constant<int, 16>{});
    return launch(places, std::integral_constant<int, 64>{});
  };
  if (top_k <= 2) return with_lanes(std::integral_constant<int, 2>{});
  if (top_k <= 4) return with_lanes(std::integral_constant<int, 4>{});
  if (top_k <= 8) return with_lanes(std::integral_constant<int, 8>{});
  return with_lanes(std::integral_constant<int, RT_MAX_CHOICES>{});
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
