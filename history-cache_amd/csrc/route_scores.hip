// Routing of rows to experts by scores, with a bias in the choice and groups of experts, and its gradient:
//
//   s = sigma(l) or softmax(l);  c = s + bias;  a group's rank: the sum of its two largest c;  the top_group best groups stay open
//   chosen: the top_k largest c in open groups, ties to the lowest index;  w = scale * s / (normalize ? sum of the chosen s : 1)
//   S = sum of the chosen s, t = scale sum_j s[j] g[j] / S
//   sigmoid:  dl[chosen j] = (normalize ? (scale g[j] - t) / S : scale g[j]) s[j] (1 - s[j])
//   softmax:  dl[chosen j] = s[j] / S (scale g[j] - t) (normalize);  dl[e] = s[e] ((e chosen ? scale g : 0) - t S)
//
// The bias keeps experts evenly loaded and is no part of the weights; a logit or a bias of -inf closes an expert.  Which of two sums
// is larger is decided in fp64: in fp32 one row in some ten thousand would go to another expert than by the formula.  Without a
// bias experts are compared by their logits, with which the score rises.
//
// Forward: a wave takes 64 / L rows.  It reads them whole and puts what is compared (c, or l without a bias) into LDS as fp32; each row
// is then gone through by L lanes, which hold the K + 1 largest of their share sorted in registers: a number's lowest bits make way for
// the expert's index, and a new one moves into the list by one median a place.  What a lane has found gets its lost bits back, is
// sorted by them and then the index, and put together with what the row's other lanes have.
// Such a choice is right where nothing near stands against it.  c in fp32 is off by up to 2^-22 and half a unit of |c|: where neighbours in
// the list, or the last open and the first closed group (by the larger of the numbers that they are sums of), are nearer than twice that and
// do not come from equal numbers, the wave decides the row again in fp64, all lanes on it.  Where the first outside the list is near by
// the bits that were kept, it is counted how many are that near by all bits.
// Bound by its vector instructions first: 500 009 rows of 64 bf16 logits to four experts 46 us for 96 MB, 1 255 instructions a wave of 32
// rows, that is 32 logits a lane: for reading logits and making scores, for the lists (K + 1 medians a logit and the index's bits), for
// joining them and for the weights of what is chosen; at one a SIMD every four cycles they are 32 of the 46 us.  With sorted lists of fp64
// keys 50, with insertion into unsorted ones 106.  65 537 rows of 256 fp32 in groups to eight 48 us for 75 MB (2 129 a wave of eight rows,
// 28 of the 48); 200 003 rows of 60 by softmax, in groups, to six 40 (2 505 a wave of 32, 26 of the 40).  Eight rows of 256 9.2: some 2 000
// instructions one after the other, which come from memory.  A whole fp64 pass over every row: 125 and 173.
// Lists have 2, 4, 8 or 32 places, so that from nine choices on a row pays for 32: 500 009 rows of 64 to eight experts 65 us, to nine 160,
// to 32 245; 65 537 of 256 38, 87 and 128; 30 000 of 1 024 80, 182 and 250.
// Backward: 23 us for 96 MB and 20 for 75 (the logits are not read: what is chosen is handed over), 139 and 160 vector instructions a wave;
// the softmax's own, which goes by the weights and needs no exponential, 54 and 16.5 us for the same 96 MB.
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
  uint32_t low;            // the bits that an index takes, and what they leave of a number's differences
  float lost;
  int piece;               // logits that are read at once
  bool softmax, normalize;
};

__device__ __forceinline__ int64_t rs_bits(double v) { return __builtin_bit_cast(int64_t, v); }
__device__ __forceinline__ double rs_double(int64_t v) { return __builtin_bit_cast(double, v); }
// What is compared lies between these as fp32, so that it stays a number when its ten lowest bits are an index: NaN and infinity as
// the largest number; a closed expert below the lowest of the others.  (Logits within 2^-12 of fp32's lowest number count as one.)
constexpr float RS_MOST = 0x1.fffffep+127f, RS_LEAST = -0x1.ffep+127f, RS_SHUT = -0x1.fffffep+127f;
__device__ __forceinline__ bool rs_shut(float c) { return c < -0x1.fffp+127f; }

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
    const float b = a.bias != nullptr ? a.bias[e] : 0.f;
    key[e] = rt_masked(l) || rt_masked(b) ? RS_CLOSED : rs_order(score(l) + (double)b);
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

// The N largest keys of the row's lanes, sorted, and the largest of the others.
template <int N>
struct rs_list {
  double t[N], out;
  __device__ __forceinline__ void sort() {
    rt_sort(t, [](double &x, double &y) { rs_in_order(x, y); });
  }
  // `out` to its place among t
  __device__ __forceinline__ void settle() {
#pragma unroll
    for (int j = 0; j < N; ++j) rs_in_order(t[j], out);
  }
  // the lists of L lanes as one, in each of them: two sorted lists that meet the other way round leave the larger half in two runs
  template <int L, int D = 1>
  __device__ __forceinline__ void join() {
    if constexpr (D < L) {
      double o[N];
#pragma unroll
      for (int j = 0; j < N; ++j) o[j] = rs_double(hc_other<D>(rs_bits(t[j])));
      out = __builtin_fmax(out, rs_double(hc_other<D>(rs_bits(out))));
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const double mine = t[j], other = o[N - 1 - j];
        t[j] = __builtin_fmax(mine, other);
        out = __builtin_fmax(out, __builtin_fmin(mine, other));
      }
#pragma unroll
      for (int d = N / 2; d >= 1; d /= 2)
#pragma unroll
        for (int i = 0; i < N; ++i)
          if ((i & d) == 0) rs_in_order(t[i], t[i + d]);
      join<L, 2 * D>();
    }
  }
};

// The larger two of the pairs that L lanes have.
template <int L, int D = 1>
__device__ __forceinline__ void rs_join_two(float &first, float &second) {
  if constexpr (D < L) {
    const float f = hc_other<D>(first), s = hc_other<D>(second);
    second = __builtin_amdgcn_fmed3f(first, f, fmaxf(second, s));
    first = fmaxf(first, f);
    rs_join_two<L, 2 * D>(first, second);
  }
}

// exp(x) by the instruction, x <= 0: off by 2^-23 and |x| 2^-23 of itself.  1 / (1 + exp(-l)) by the instructions, within 2^-22.
__device__ __forceinline__ float rs_near_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }
__device__ __forceinline__ float rs_near_sigma(float l) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(l * -1.44269504f));
}

// s = 1 / (1 + exp(-l)) on the scale exp(-base), base <= 0, l <= base or base = 0; and 1 - s.  What is divided by its sum is taken on the scale of the largest logit, so that scores which 32 bits do not hold (l < -87) still have their shares.
__device__ __forceinline__ float rs_sigma(float l, float base, float &rest) {
  const float x = expf(-fabsf(l)), y = 1.f + x, near = __builtin_amdgcn_rcpf(y);
  const float q = __builtin_fmaf(__builtin_fmaf(-y, near, 1.f), near, near);               // (1 / y, right but for the last bit)
  rest = l >= 0.f ? x * q : q;
  return l >= 0.f ? q : (base < 0.f ? expf(l - base) : x) * q;
}
__device__ __forceinline__ float rs_base(float largest) { return fminf(largest, 0.f); }
// Scores of less than exp of this are 0, as they soon are in 64 bits.
constexpr float RS_NOTHING = -700.f;

// What is compared, as it lies in LDS: of a logit or a bias; of a sum that cannot be too small; of a logit and a bias in LDS.
__device__ __forceinline__ float rs_plain(float l) {
  return rt_masked(l) ? RS_SHUT : fmaxf(fminf(l + 0.f, RS_MOST), RS_LEAST);
}
__device__ __forceinline__ float rs_choice(float l, float bias) {
  const float c = fminf(rs_near_sigma(l) + bias, RS_MOST);
  return rt_masked(l) || rs_shut(bias) ? RS_SHUT : c;          // (beside a closed one's NaN, too)
}

// Rows r0 .. r0 + rows into LDS: c where the score is a logit's own and there is a bias, l otherwise.
template <typename T, int PIECE>
__device__ __forceinline__ void rs_stage(const RsArgs &a, int64_t r0, int rows, float *s, const float *bias) {
  constexpr int AT_ONCE = 4;
  const int lane = hc_lane();
  const T *from = static_cast<const T *>(a.logits) + r0 * a.E;
  const bool make = a.bias != nullptr && !a.softmax;
  if constexpr (PIECE > 1) {
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
      if (a.E + x % 4 < 4 * a.quads) s[x / 4 * a.stride + a.E + x % 4] = RS_SHUT;
  }
}

// Calls f(four values, index of the first) for the elements from .. to of a row in LDS that lane `sub` of L takes; behind `to`: shut.
template <int L, typename F>
__device__ __forceinline__ void rs_each(const float *row, int from, int to, int sub, bool by_four, F &&f) {
  if (by_four) {
    for (int e = from + 4 * sub; e < to; e += 4 * L) f(*reinterpret_cast<const float4 *>(row + e), e);
  } else {
    for (int e = from + 4 * sub; e < to; e += 4 * L)
      f(make_float4(row[e], e + 1 < to ? row[e + 1] : RS_SHUT, e + 2 < to ? row[e + 2] : RS_SHUT, e + 3 < to ? row[e + 3] : RS_SHUT),
        e);
  }
}

// K: places for winners, k <= K; L: lanes a row.
template <int K, int L>
__global__ __launch_bounds__(HC_WAVE) void rs_forward(RsArgs a) {
  // rows, the groups' ranks of each, the bias
  extern __shared__ __attribute__((aligned(16))) float s_all[];
  constexpr int ROWS = HC_WAVE / L, OWN = (K + L - 1) / L;
  const int lane = hc_lane(), sub = lane % L, mine = lane / L;
  const int64_t r0 = (int64_t)blockIdx.x * ROWS;
  const int rows = a.n - r0 < ROWS ? (int)(a.n - r0) : ROWS;
  const bool live = mine < rows;
  const int64_t r = r0 + (live ? mine : 0);
  const bool exact = a.bias == nullptr;              // what is compared are logits
  float *bias = s_all + ROWS * (a.stride + a.rank_stride);
  if (!exact) {
    for (int e = lane; e < a.E; e += HC_WAVE) bias[e] = rs_plain(a.bias[e]);
    rt_in_order();
  }
  const auto stage = [&](auto type) {
    typedef decltype(type) T;
    if (a.piece == 8) rs_stage<T, sizeof(T) == 2 ? 8 : 4>(a, r0, rows, s_all, bias);
    else if (a.piece >= 4) rs_stage<T, 4>(a, r0, rows, s_all, bias);
    else rs_stage<T, 1>(a, r0, rows, s_all, bias);
  };
  if (a.dtype == HC_F32) stage(float{});
  else if (a.dtype == HC_F16) stage(__half{});
  else stage(__hip_bfloat16{});
  rt_in_order();
  float *row = s_all + (live ? mine : 0) * a.stride;
  float top = RS_SHUT, all = 0.f;
  bool near = false, no_number = false;              // too near for fp32; a softmax with an infinity or a NaN in it
  if (a.softmax) {
    rs_each<L>(row, 0, 4 * a.quads, sub, true, [&](float4 l, int) { top = fmaxf(top, fmaxf(fmaxf(l.x, l.y), fmaxf(l.z, l.w))); });
    top = hc_join<L>(top, [](float x, float y) { return fmaxf(x, y); });
    // (a closed expert lies so far below every other that its exponential is 0)
    double sum = 0.0;
    rs_each<L>(row, 0, 4 * a.quads, sub, true, [&](float4 l, int) {
      sum += ((double)rs_near_exp(l.x - top) + (double)rs_near_exp(l.y - top)) +
             ((double)rs_near_exp(l.z - top) + (double)rs_near_exp(l.w - top));
    });
    sum = rs_double(hc_join<L>(rs_bits(sum), [](int64_t x, int64_t y) { return rs_bits(rs_double(x) + rs_double(y)); }));
    all = (float)sum;
    if (__ballot(top >= RS_MOST) != 0) {
      int bad = 0;
      for (int e = sub; e < a.E; e += L) bad |= rs_logit(a, r * a.E + e) < __builtin_inff() ? 0 : 1;
      no_number = hc_join<L>(bad, [](int x, int y) { return x | y; }) != 0;
      near = no_number && !exact;
    }
    if (!exact) {
      rt_in_order();
      if (live)
        for (int e = sub; e < a.E; e += L) {
          const float l = row[e];
          row[e] = rs_shut(l) ? l : fminf(expf(l - top) / all + bias[e], RS_MOST);
        }
      rt_in_order();
    }
  }
  uint64_t open = ~0ull;
  const bool by_four = a.per_group % 4 == 0;
  if (a.groups > 1) {
    float *rank = s_all + ROWS * a.stride + mine * a.rank_stride;
    float size = 0.f;                                // of the summands, whose errors a sum has
    for (int g = 0; g < a.groups; ++g) {
      float first = RS_SHUT, second = RS_SHUT;
      const auto more = [&](float c) {
        second = __builtin_amdgcn_fmed3f(first, second, c);
        first = fmaxf(first, c);
      };
      rs_each<L>(row, g * a.per_group, (g + 1) * a.per_group, sub, by_four, [&](float4 c, int) {
        more(c.x);
        more(c.y);
        more(c.z);
        more(c.w);
      });
      rs_join_two<L>(first, second);
      near = near || first >= RS_MOST;               // (infinite, or no number)
      size = fmaxf(size, fmaxf(rs_shut(first) ? 0.f : fabsf(first), rs_shut(second) ? 0.f : fabsf(second)));
      if (exact && !rs_shut(first)) {
        first = a.softmax ? rs_near_exp(first - top) : rs_near_sigma(first);
        second = rs_shut(second) ? second : a.softmax ? rs_near_exp(second - top) : rs_near_sigma(second);
      }
      if (sub == 0) rank[g] = rs_shut(second) ? first : first + second;
    }
    rt_in_order();
    // the last open group and the first closed one
    float least = RS_MOST, most = RS_SHUT;
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
    // (scores below 2^-126 are 0 to the instructions)
    const float off = exact ? 0x1p-15f * fmaxf(fabsf(least), 0x1p-100f) : 0x1p-19f * (1.f + size);
    near = near || (!rs_shut(most) && !(least - most > off));
  }
  // f for the row's open elements that this lane takes
  const auto each_open = [&](auto &&f) {
    if (a.groups > 1) {
      uint64_t left = open;
      for (int t = 0; t < a.top_group; ++t) {
        const int g = left != 0 ? __builtin_ctzll(left) : 0;
        left &= left - 1;
        rs_each<L>(row, g * a.per_group, (g + 1) * a.per_group, sub, by_four, f);
      }
    } else {
      rs_each<L>(row, 0, 4 * a.quads, sub, true, f);
    }
  };
  rs_list<K> list;
  {
    float t[K + 1];
#pragma unroll
    for (int j = 0; j <= K; ++j) t[j] = RS_SHUT;
    const uint32_t low = a.low;
    // SIGNED: the lower of two indexes makes a negative number the larger one, too (sums below 0 are left to the look at what is near)
    const auto fill = [&](auto signed_) {
      const auto more = [&](float c, int e) {
        const uint32_t b = __float_as_uint(c), turn = decltype(signed_)::value ? (uint32_t)((int32_t)b >> 31) & low : 0u;
        const float x = __uint_as_float((b & ~low) | ((low - (uint32_t)e) ^ turn));
#pragma unroll
        for (int j = K; j >= 1; --j) t[j] = __builtin_amdgcn_fmed3f(t[j - 1], t[j], x);
        t[0] = __builtin_amdgcn_fmed3f(t[0], x, __builtin_inff());
      };
      each_open([&](float4 c, int e) {
        more(c.x, e);
        more(c.y, e + 1);
        more(c.z, e + 2);
        more(c.w, e + 3);
      });
    };
    if (exact) fill(std::true_type{});
    else fill(std::false_type{});
    // (indexes behind the row's end are those of shut places, of which the list's first ones are some as well)
    const auto whole = [&](float x) {
      const uint32_t b = __float_as_uint(x), turn = exact ? (uint32_t)((int32_t)b >> 31) & low : 0u;
      const int e = (int)(low - ((b & low) ^ turn));
      const float c = row[e < a.stride ? e : 0];
      return rs_shut(x) ? rs_key(RS_SHUT, 0) : rs_key(c, e);
    };
#pragma unroll
    for (int j = 0; j < K; ++j) list.t[j] = whole(t[j]);
    list.out = whole(t[K]);
  }
  list.sort();
  list.settle();
  list.template join<L>();
  if (rs_key_value(list.t[1]) >= RS_MOST) near = true;                 // (two that are infinite or no numbers)
  if (!exact || a.dtype == HC_F32) {
    // l and bias of two experts
    const auto equal = [&](double x, double y) {
      const int i = rs_key_index(x), j = rs_key_index(y);
      return rs_logit(a, r * a.E + i) == rs_logit(a, r * a.E + j) && (exact || bias[i] == bias[j]);
    };
    if (!exact) {
#pragma unroll
      for (int j = 0; j + 1 < K; ++j) {
        const float c = rs_key_value(list.t[j]), d = rs_key_value(list.t[j + 1]);
        // (of equal numbers the lower index is the right one)
        if (j + 1 < a.k && !rs_shut(d) && !(c - d > 0x1p-20f * (1.f + fabsf(c)))) near = near || !equal(list.t[j], list.t[j + 1]);
      }
    }
    double last = list.t[0], next = list.out;
#pragma unroll
    for (int j = 1; j < K; ++j) {
      if (j == a.k) next = list.t[j];
      if (j < a.k) last = list.t[j];
    }
    const float c = rs_key_value(last), d = rs_key_value(next), off = exact ? 0.f : 0x1p-20f * (1.f + fabsf(c));
    const bool count = !near && !rs_shut(d) && !(c - d > off + a.lost * fmaxf(fabsf(c), 0x1p-126f));
    if (__ballot(count) != 0) {
      // with logits the last winner's place in the row, otherwise how many are not clearly behind it
      int there = 0;
      const int at = exact ? rs_key_index(last) : a.E;
      const float from = c - off;
      each_open([&](float4 v, int e) {
        there += v.x > from || (v.x == from && e <= at) ? 1 : 0;
        there += v.y > from || (v.y == from && e + 1 <= at) ? 1 : 0;
        there += v.z > from || (v.z == from && e + 2 <= at) ? 1 : 0;
        there += v.w > from || (v.w == from && e + 3 <= at) ? 1 : 0;
      });
      there = hc_join<L>(there, [](int x, int y) { return x + y; });
      if (count) near = there > a.k && (exact || !(there == a.k + 1 && equal(last, next)));
    }
  }
  // this lane's winners
  int won[OWN];
#pragma unroll
  for (int u = 0; u < OWN; ++u) {
    double x = list.t[u * L];
#pragma unroll
    for (int d = 1; d < L; ++d)
      if (u * L + d < K && sub == d) x = list.t[u * L + d];
    won[u] = u * L + sub < a.k && !rs_shut(rs_key_value(x)) ? rs_key_index(x) : -1;
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
#pragma unroll
      for (int u = 0; u < OWN; ++u)
        if (mine == row_of && u * L + sub < a.k) won[u] = found[u * L + sub];
      rt_in_order();
    }
  }
  // shares on the scale of the largest chosen; where that is nothing beside the row, or by itself, so are the weights
  float p[OWN], s[OWN], sum = 0.f, largest = -__builtin_inff();
#pragma unroll
  for (int u = 0; u < OWN; ++u) {
    p[u] = won[u] >= 0 ? rs_logit(a, r * a.E + won[u]) : 0.f;
    if (won[u] >= 0) largest = fmaxf(largest, a.softmax ? rs_plain(p[u]) : p[u]);
  }
  if (a.normalize) largest = hc_join<L>(largest, [](float x, float y) { return fmaxf(x, y); });
  const float base = a.softmax ? (a.normalize ? largest : top) : a.normalize ? rs_base(largest) : 0.f;
#pragma unroll
  for (int u = 0; u < OWN; ++u) {
    float rest;
    s[u] = won[u] < 0 ? 0.f : a.softmax ? expf(rs_plain(p[u]) - base) : rs_sigma(p[u], base, rest);
    sum += s[u];
  }
  sum = hc_join<L>(sum, [](float x, float y) { return x + y; });
  const bool nothing = a.normalize && (a.softmax ? largest - top : largest) < RS_NOTHING && sum == sum;
  if (nothing) sum = 0.f;
  if (no_number) all = sum = __builtin_nanf("");
  const float of = a.normalize ? sum : a.softmax ? all : 1.f;
  if (!live) return;
#pragma unroll
  for (int u = 0; u < OWN; ++u) {
    const int j = u * L + sub;
    if (j >= a.k) continue;
    a.expert[r * a.k + j] = won[u];
    a.weight[r * a.k + j] = won[u] < 0 || of == 0.f ? 0.f : a.scale * (s[u] / of);
    if (a.picked != nullptr) {
      // (a chosen one need not be the infinity or NaN that makes all of its row's scores NaN)
      const float kept = no_number ? __builtin_nanf("") : nothing ? -__builtin_inff() : p[u] < RS_LEAST ? RS_LEAST : p[u];
      a.picked[r * a.k + j] = won[u] >= 0 ? kept : 0.f;
    }
  }
}

struct RsGradArgs {
  const void *logits;
  const int64_t *expert;
  const float *picked, *g;
  void *grad;
  int64_t n;
  float scale;
  int E, k;
  bool softmax, normalize, whole;
};

// By the chosen logits alone, but for softmax weights as they are, which go by all of a row's.
template <typename T, int L, int V>
__global__ __launch_bounds__(HC_BLOCK) void rs_backward(RsGradArgs a) {
  // the row in LDS: what its choices bring, each from the lane that has read it; zeros elsewhere
  __shared__ __attribute__((aligned(16))) float s_row[HC_BLOCK * V];
  const int lane = (int)threadIdx.x & (L - 1);
  const int64_t r = ((int64_t)blockIdx.x * HC_BLOCK + threadIdx.x) / L;
  const bool live = r < a.n;
  const int64_t at = (live ? r : 0) * a.k;
  const auto plus = [](float x, float y) { return x + y; };
  const auto larger = [](float x, float y) { return fmaxf(x, y); };
  const bool by_row = a.softmax && !a.normalize;
  float *own = s_row + threadIdx.x * V, *row = own - lane * V;
#pragma unroll
  for (int i = 0; i < V; ++i) own[i] = 0.f;
  // a choice: its expert, what reaches its weight, its logit (the first L choices stay in registers)
  struct choice {
    int64_t e;
    float d, p;
  };
  const auto read = [&](int j) {
    choice c{-1, 0.f, 0.f};
    if (j < a.k) {
      c.e = a.expert[at + j];
      c.d = a.scale * a.g[at + j];
      if (!by_row) c.p = a.picked[at + j];
    }
    return c;
  };
  const choice mine = read(lane);
  float top = RS_SHUT;
  if (a.normalize) {
    if (mine.e >= 0) top = fmaxf(top, mine.p);
    for (int j = lane + L; j < a.k; j += L) {
      const choice c = read(j);
      if (c.e >= 0) top = fmaxf(top, c.p);
    }
    top = hc_join<L>(top, larger);
  }
  // s of a choice, normalised on the scale of the largest, and what its slope is more than s
  const float base = a.normalize ? rs_base(top) : 0.f;
  const auto score = [&](const choice &c, float &rest) {
    rest = 1.f;
    return c.e < 0 ? 0.f : a.softmax ? expf(c.p - top) : rs_sigma(c.p, base, rest);
  };
  float rest = 1.f, s = by_row ? 1.f : score(mine, rest), sum = s, inverse = 0.f, t = 0.f;
  // (a reciprocal and one correction: the share of a choice that is its row's only one is 1, and its gradient 0)
  const auto share = [&](float s) {
    const float f = s * inverse;
    return __builtin_fmaf(__builtin_fmaf(-f, sum, s), inverse, f);
  };
  if (a.normalize) {
    for (int j = lane + L; j < a.k; j += L) {
      float other;
      sum += score(read(j), other);
    }
    sum = hc_join<L>(sum, plus);
    // (the largest's own score is a half at least, and all are 0 where the weights are)
    inverse = sum == 0.f ? 0.f : __builtin_amdgcn_rcpf(sum);
    s = share(s);
    // (what reaches a weight that stands for nothing may be no number)
    t = mine.e < 0 ? 0.f : s * mine.d;
    for (int j = lane + L; j < a.k; j += L) {
      const choice c = read(j);
      float other;
      t += c.e < 0 ? 0.f : share(score(c, other)) * c.d;
    }
    t = hc_join<L>(t, plus);
  }
  rt_in_order();
  const auto bring = [&](const choice &c, float ds) {
    if (c.e >= 0 && c.e < a.E) row[c.e] = by_row ? c.d : (c.d - t) * ds;
  };
  bring(mine, s * rest);
  for (int j = lane + L; j < a.k; j += L) {
    const choice c = read(j);
    float other = 1.f, f = 1.f;
    if (!by_row) f = score(c, other);
    bring(c, (a.normalize ? share(f) : f) * other);
  }
  rt_in_order();
  float out[V];
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = own[i];
  if (by_row) {
    T v[V];
    float p[V], most = -__builtin_inff(), all = 0.f;
    rt_row<T, V>::load(static_cast<const T *>(a.logits) + (live ? r : 0) * a.E, lane * V, a.E, a.whole, v);
#pragma unroll
    for (int i = 0; i < V; ++i) most = fmaxf(most, hc_to_f32<T>(v[i]));
    most = hc_join<L>(most, larger);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float f = hc_to_f32<T>(v[i]);
      p[i] = rt_masked(f) ? 0.f : expf(f - most);
      all += p[i];
    }
    all = hc_join<L>(all, plus);
    float inner = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      p[i] = all == 0.f ? 0.f : p[i] / all;
      inner += p[i] * out[i];
    }
    inner = hc_join<L>(inner, plus);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = p[i] * (out[i] - inner);
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
           top_group == num_group ? 1 : (int)num_group, (int)(E / num_group), (int)top_group, 0, 0, 0, 0, 0.f, 1, score != RS_SIGMOID,
           normalize != 0};
  a.low = 15;
  while (a.low + 1 < (uint32_t)(E + 3) / 4 * 4) a.low = 2 * a.low + 1;
  a.lost = (float)(a.low + 1) * 0x1p-22f;
  if (dtype == HC_F32) a.piece = rt_row<float, 4>::whole(logits, E) ? 4 : 1;
  else a.piece = rt_row<__half, 8>::whole(logits, E) ? 8 : rt_row<__half, 4>::whole(logits, E) ? 4 : 1;
  a.quads = (int)((E + 3) / 4);
  const auto launch = [&](auto places, auto lanes) {
    constexpr int L = decltype(lanes)::value;
    const int64_t blocks = (n + HC_WAVE / L - 1) / (HC_WAVE / L);
    if (blocks > (int64_t)(0xffffffffu / HC_WAVE)) return (int)HC_EUNSUPPORTED;
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
  // Lanes a row: as few as leave a compute unit enough waves beside their rows in LDS (9.5 KB a wave), and twice as many where that makes
  // fewer waves than there are SIMDs.  (Twice as many again are 0.4 to 1 us faster up to 16 000 rows of 64 and 2 slower at 30 000; with 256
  // experts 0.6 slower at 64 rows, 1 to 6 faster at 1 000, 3 to 6 slower from 4 000 on: no third set of kernels for that.)  Us by 1 / 2 / 4 /
  // 8 lanes: 500 009 rows of 64 50 / 43 / 47, 30 000 15 / 11 / 9.3 / 9.3, 250 8.7 / 6.0 / 4.5 / 4.2; by 4 / 8 / 16 / 32: 65 537 rows of 256 in
  // groups 51 / 48 / 65, 8 000 23 / 21 / 21 / 27, 250 14.5 / 10.7 / 10.2 / 9.3; by 16 / 32 / 64: 30 000 rows of 1 024 78 / 79 / 94, 250
  // 14.6 / 10.5 / 8.8.
  const auto with_lanes = [&](auto places) {
    const int least = E <= 64 ? 2 : E <= 256 ? 8 : 32;
    const bool few = n * least < 64 * 1024;
    if (least == 2) return few ? launch(places, std::integral_constant<int, 4>{}) : launch(places, std::integral_constant<int, 2>{});
    if (least == 8) return few ? launch(places, std::integral_constant<int, 16>{}) : launch(places, std::integral_constant<int, 8>{});
    return few ? launch(places, std::integral_constant<int, 64>{}) : launch(places, std::integral_constant<int, 32>{});
  };
  if (top_k <= 2) return with_lanes(std::integral_constant<int, 2>{});
  if (top_k <= 4) return with_lanes(std::integral_constant<int, 4>{});
  if (top_k <= 8) return with_lanes(std::integral_constant<int, 8>{});
  return with_lanes(std::integral_constant<int, RT_MAX_CHOICES>{});
}

extern "C" int hc_route_scores_grad(const void *logits, int dtype, int64_t n, int64_t E, int64_t top_k, int score, int normalize,
                                    float scale, const int64_t *expert, const float *picked, const float *grad_weight,
                                    void *grad_logits, void *stream) {
  if (const int rc = rs_sizes(n, E, top_k, score, scale)) return rc;
  if (n == 0) return dtype >= HC_F32 && dtype <= HC_BF16 ? HC_OK : HC_EDTYPE;
  HC_REQUIRE((score != RS_SIGMOID && !normalize ? logits != nullptr : picked != nullptr) && expert && grad_weight && grad_logits);
  return rt_with_type(dtype, [&](auto type) {
    typedef decltype(type) T;
    return rt_with_shape((int)E, [&](auto lanes, auto each) {
      constexpr int L = decltype(lanes)::value, V = decltype(each)::value;
      const int64_t blocks = (n + HC_BLOCK / L - 1) / (HC_BLOCK / L);
      if (!hc_grid_ok(blocks)) return (int)HC_EUNSUPPORTED;
      const RsGradArgs a{logits, expert, picked, grad_weight, grad_logits, n, scale, (int)E, (int)top_k,
                         score != RS_SIGMOID, normalize != 0,
                         rt_row<T, V>::whole(logits, E) && rt_row<T, V>::whole(grad_logits, E)};
      rs_backward<T, L, V><<<dim3((unsigned)blocks), dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(a);
      return hc_launch_status();
    });
  });
}
