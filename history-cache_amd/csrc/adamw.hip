// An AdamW step over many tensors in one launch, its states in 32 or in 8 bits:
//
//   t += 1;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g g
//   p = p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in fp32, each operation rounded, the powers in fp64.  t is the tensor's own and lies on the device, so that a recording can be
// replayed; the block that ends last counts it up.  A parameter of 16 bits may have a copy in fp32 that takes the step (an update
// below half a unit of the parameter would be lost).
//
// 8 bits: m and r = sqrt(v) as numbers of four bits of exponent; m has a sign and three bits of mantissa, r, which has none, four.
// 128 adjacent elements share the exponent E (one byte, as fp32's biased exponent) of their largest magnitude rounded to that
// mantissa.  Elements differ by orders of magnitude, and an update goes by m / r: equal steps would lose the small ones
// altogether, a mantissa keeps each within 1/16 (r: 1/32) down to 2^-14 of the largest, and 2^-18 (r: 2^-19) of that below.  r is
// rounded up from zero: an element whose r was lost would move by m / eps.  (Scaled by 2^(15 - E) a number's upper bits are
// its code, subnormal ones included.)  E = 0: zeros, the largest is below fp32's normal numbers.  E = 255: a group that held an
// infinity or a NaN, all of which reads back as NaN.
//
// A code is the nearest one, or (HC_ADAMW_RANDOM) one of the two that a number lies between, the upper one as often as the number lies
// nearer to it.  The nearest one is right for one step from given moments; over many it stops r, which moves by (1 - b2) / 2 of itself a
// step, far less than half a code: at b2 = 0.999 and gradients that stay as they are it ends at 0.13 to 0.5 of the right one, and
// never falls again.  At random a number is kept in the mean: r's mean over elements stays within 1 % of the right one at any b2, an
// element's own within 10 % (one standard deviation; a step's is half a percent, and they add up over the steps that v remembers).  What
// is random is a hash of the element's place in its tensor and the tensor's count, so that a step that is made again, in a
// recording, or in another launch is the same.
//
// A block takes pieces of 2 048 elements of the tensors' concatenation, eight a lane; sixteen lanes share a group.  Every element is
// read and written once, which bounds large calls: 50.3 M elements of fp32 (us and TB/s) with 8 bits 166 (4.9), 32 bits 278 (5.1), of
// bf16 with 8 bits 103 to 108 (4.8), with a copy in fp32 168 (4.8), 32 bits 219 (5.0), with a copy 284 (5.0); rounded at random, fifteen
// operations an element more, the same.  torch's copy of 4 GiB reaches 4.8 TB/s, of 256 MiB 5.4.  Eight
// small tensors take 6.6 us: their counts, the powers of the rates in 64 bits, a memory's latency for the elements and one for
// the arrival.  Non-temporal stores: no difference.
#include "packed_rows.h"

namespace {

constexpr int AW_MAX = 48;                   // tensors a launch: 3.4 KB of arguments
constexpr int AW_GROUP = 128;
constexpr int AW_LANES = AW_GROUP / PK_EACH;
constexpr int AW_PIECE = HC_BLOCK * PK_EACH;
constexpr int AW_BLOCKS = 2048;              // eight blocks a compute unit; more pieces: a block takes several

struct AwTensor {
  void *p;
  const void *g;
  void *m, *v;
  uint8_t *scale;          // [2, groups]: E of m, E of r
  float *master;
  int64_t *step;           // the count; a counter of blocks, zero between calls
  int64_t n;
};

struct AwArgs {
  AwTensor t[AW_MAX];
  uint32_t first[AW_MAX + 1];                // number of the first piece of every tensor
  int count;
  double lr, b1, b2, decay;
  const float *lr_dev;
  float eps;
};

__device__ __forceinline__ double aw_power(double b, int64_t t) {
  double r = 1.0;
  for (; t > 0; t >>= 1) {
    if (t & 1) r *= b;
    b *= b;
  }
  return r;
}

// Two rounds of an odd factor (the golden section's, the circle number's digits) and the upper half folded into the lower one: a change of
// one bit changes every other in about half of all cases.
__device__ __forceinline__ uint32_t aw_mix(uint32_t x) {
  x = (x ^ x >> 16) * 0x9e3779b1u;
  x = (x ^ x >> 15) * 0x85a308d3u;
  return x ^ x >> 16;
}

// What a tensor's elements share.
struct AwFactors {
  float keep, size, lift;
  uint32_t key;                              // of what is random in this step
  __device__ __forceinline__ void work_out(const AwArgs &a, int64_t count) {
    const double lr = a.lr_dev != nullptr ? (double)*a.lr_dev : a.lr;
    keep = (float)(1.0 - lr * a.decay);
    size = (float)(lr / (1.0 - aw_power(a.b1, count)));
    lift = (float)(1.0 / sqrt(1.0 - aw_power(a.b2, count)));
    key = aw_mix(aw_mix((uint32_t)count) + (uint32_t)((uint64_t)count >> 32) * 0x9e3779b1u + 0x243f6a88u);
  }
};

// sqrt(x) for x >= 0, correctly rounded from 2^-96 up (below within a unit in the last place): the instruction's result or one of its
// neighbours.
__device__ __forceinline__ float aw_sqrt(float x) {
  const float y = __builtin_amdgcn_sqrtf(x);
  const float down = __uint_as_float(__float_as_uint(y) - 1u), up = __uint_as_float(__float_as_uint(y) + 1u);
  const float r = __builtin_fmaf(-down, y, x) <= 0.f ? down : y;
  return __builtin_fmaf(-up, y, x) > 0.f ? up : r;
}

// ---- numbers of 8 bits: MAN bits of mantissa (3: with a sign, 4: without)
// A group of E = 255 is NaN: that comes in by the sum of its first operation (aw_poison).
__device__ __forceinline__ float aw_poison(uint32_t E) { return E == 255u ? __builtin_nanf("") : 0.f; }

template <int MAN>
__device__ __forceinline__ void aw_decode(const uint32_t (&w)[2], uint32_t E, float (&v)[PK_EACH]) {
#pragma unroll
  for (int i = 0; i < PK_EACH; ++i) {
    const uint32_t u = w[i / 4], at = 8 * (i % 4);
    const uint32_t b = MAN == 3 ? (uint32_t)((int32_t)(u << (24 - at)) >> 24 << 20) & 0x87f00000u : (u >> at & 0xffu) << 19;
    v[i] = __builtin_amdgcn_ldexpf(__uint_as_float(b), (int)E - 15);
  }
}

// Adds half a unit of MAN bits of mantissa to fp32 bits, a little less where that breaks a tie the even way.  RANDOM: what half of
// a random word (its lower one for three bits, its upper one for four) is of a unit, 2^-17 more, so that a code's own number stays.
template <int MAN, bool RANDOM>
__device__ __forceinline__ uint32_t aw_round(uint32_t b, uint32_t random) {
  if constexpr (RANDOM) return b + (MAN == 3 ? (random & 0xffffu) << 4 | 8u : (random >> 16) << 3 | 4u);
  return b + (1u << (22 - MAN)) - 1u + (b >> (23 - MAN) & 1u);
}

// The E of the group that AW_LANES lanes hold, and this lane's codes.
template <int MAN, bool RANDOM>
__device__ __forceinline__ uint32_t aw_encode(const float (&v)[PK_EACH], const uint32_t (&random)[PK_EACH], uint32_t (&w)[2]) {
  uint32_t most = 0, least = 0xffffffffu;    // (of magnitudes' bits; the least one's that is not 0, less 1)
#pragma unroll
  for (int i = 0; i < PK_EACH; ++i) {
    uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    if constexpr (RANDOM) b = aw_round<MAN, true>(b, random[i]);       // (which of them is the largest goes by what they become)
    else least = b - 1u < least ? b - 1u : least;
    most = b > most ? b : most;
  }
  most = hc_join<AW_LANES>(most, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
  const uint32_t top = (RANDOM ? most : aw_round<MAN, false>(most, 0)) >> 23, E = top > 255u ? 255u : top;
  uint32_t c[PK_EACH];                       // the code in the upper byte
#pragma unroll
  for (int i = 0; i < PK_EACH; ++i) {
    uint32_t b = __float_as_uint(__builtin_amdgcn_ldexpf(v[i], 15 - (int)E));
    if constexpr (MAN == 3) {
      b = aw_round<3, RANDOM>(b, random[i]);
      c[i] = (b & 0x80000000u) | (b << 4 & 0x7fffffffu);
    } else {
      // (a root that is not 0 is above 2^-75)
      const uint32_t lowest = __float_as_uint(v[i]) < 1u << 19 ? __float_as_uint(v[i]) : 1u << 19;
      b = b > lowest ? b : lowest;
      c[i] = aw_round<4, RANDOM>(b, random[i]) << 5;
    }
  }
  if constexpr (!RANDOM) {
    // Scaled down to below fp32's normal numbers one has been rounded before it is rounded to a code, and may have become a tie: those
    // are taken in units of the smallest code instead, which are exact.
    if (__any(E > 15u && least < ((E - 14u) << 23) - 1u)) {
#pragma unroll
      for (int i = 0; i < PK_EACH; ++i) {
        const float u = __builtin_amdgcn_ldexpf(fabsf(v[i]), 141 + MAN - (int)E);
        uint32_t code = (uint32_t)__builtin_rintf(u);
        if (MAN == 4 && v[i] > 0.f && code == 0) code = 1;
        if (u < (float)(1 << MAN)) c[i] = MAN == 3 ? (__float_as_uint(v[i]) & 0x80000000u) | code << 24 : code << 24;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // the upper bytes of four words
    const uint32_t lo = __builtin_amdgcn_perm(c[4 * i + 1], c[4 * i], 0x00000703u);
    const uint32_t hi = __builtin_amdgcn_perm(c[4 * i + 3], c[4 * i + 2], 0x07030000u);
    w[i] = (lo & 0xffffu) | (hi & 0xffff0000u);
  }
  if (E == 0 || E == 255u) w[0] = w[1] = 0;
  return E;
}

__device__ __forceinline__ void aw_load_codes(const void *p, int64_t at, int valid, uint32_t (&w)[2]) {
  const char *q = static_cast<const char *>(p) + at;
  if (valid >= PK_EACH) {
    const pk_codes c = *reinterpret_cast<const pk_codes *>(q);
    w[0] = c.w[0];
    w[1] = c.w[1];
  } else {
    pk_load_tail<1>(q, valid, w);
  }
}

__device__ __forceinline__ void aw_store_codes(void *p, int64_t at, int valid, const uint32_t (&w)[2]) {
  char *q = static_cast<char *>(p) + at;
  if (valid >= PK_EACH) *reinterpret_cast<pk_codes *>(q) = pk_codes{{w[0], w[1]}};
  else if (valid > 0) pk_store_tail<1>(q, valid, w);
}

// RANDOM: states in 8 bits are rounded at random.
template <typename T, int BITS, bool MASTER, bool RANDOM>
__global__ __launch_bounds__(HC_BLOCK) void aw_step(AwArgs a) {
  const float b1 = (float)a.b1, c1 = (float)(1.0 - a.b1), b2 = (float)a.b2, c2 = (float)(1.0 - a.b2);
  __shared__ AwFactors s_factor[AW_MAX];
  const bool counts = (int)threadIdx.x < a.count;
  const int64_t count = counts ? *a.t[threadIdx.x].step + 1 : 0;
  // s_factor is worked out while a block's first piece is on its way where that costs nothing: with states in 8 bits, whose pieces
  // have more operations, the loop without it is faster (50 M elements of bf16 104 us against 118; eight small tensors in 32 bits
  // 6.8 against 6.5).
  bool known = false;
  const auto work_out = [&] {
    if (counts) s_factor[threadIdx.x].work_out(a, count);
    __syncthreads();
    known = true;
  };
  if constexpr (BITS == 8) work_out();
  uint32_t piece = blockIdx.x;
  const uint32_t pieces = a.first[a.count];
  for (int i = 0; piece < pieces;) {
    while (piece >= a.first[i + 1]) ++i;
    const AwTensor t = a.t[i];
    AwFactors f;
    if (BITS == 8 || known) f = s_factor[i];
    const int64_t groups = (t.n + AW_GROUP - 1) / AW_GROUP;
    const uint32_t first = a.first[i], end = a.first[i + 1];
    for (; piece < end; piece += gridDim.x) {
      const int64_t at = (int64_t)(piece - first) * AW_PIECE + (int64_t)threadIdx.x * PK_EACH;
      const int64_t left = t.n - at;
      const int valid = left >= PK_EACH ? PK_EACH : left > 0 ? (int)left : 0;
      float p[PK_EACH], g[PK_EACH], m[PK_EACH], v[PK_EACH];
      pk_row<T>::load(static_cast<const T *>(t.g) + at, valid, g);
      if constexpr (MASTER) pk_row<float>::load(t.master + at, valid, p);
      else pk_row<T>::load(static_cast<const T *>(t.p) + at, valid, p);
      if constexpr (BITS == 8) {
        uint32_t wm[2], wv[2], Em = 0, Ev = 0;
        aw_load_codes(t.m, at, valid, wm);
        aw_load_codes(t.v, at, valid, wv);
        if (valid > 0) Em = t.scale[at / AW_GROUP], Ev = t.scale[groups + at / AW_GROUP];
        aw_decode<3>(wm, Em, m);
        aw_decode<4>(wv, Ev, v);
        const float nan_m = aw_poison(Em), nan_v = aw_poison(Ev);
#pragma unroll
        for (int k = 0; k < PK_EACH; ++k) {
          m[k] = __builtin_fmaf(b1, m[k], nan_m);
          v[k] = b2 * __builtin_fmaf(v[k], v[k], nan_v);
        }
      } else {
        pk_row<float>::load(static_cast<const float *>(t.m) + at, valid, m);
        pk_row<float>::load(static_cast<const float *>(t.v) + at, valid, v);
#pragma unroll
        for (int k = 0; k < PK_EACH; ++k) m[k] = b1 * m[k], v[k] = b2 * v[k];
      }
      if constexpr (BITS == 32) {
        if (!known) {
          work_out();
          f = s_factor[i];
        }
      }
      float r[PK_EACH];
#pragma unroll
      for (int k = 0; k < PK_EACH; ++k) {
        m[k] = m[k] + c1 * g[k];
        v[k] = v[k] + c2 * g[k] * g[k];
        r[k] = aw_sqrt(v[k]);
        // (the reciprocal is off by a unit in the last place: of a step that is some thousandth of p)
        p[k] = p[k] * f.keep - f.size * (m[k] * __builtin_amdgcn_rcpf(r[k] * f.lift + a.eps));
      }
      if constexpr (MASTER) pk_row<float>::store(t.master + at, valid, p);
      pk_row<T>::store(static_cast<T *>(t.p) + at, valid, p);
      if constexpr (BITS == 8) {
        if (valid < PK_EACH) {
#pragma unroll
          for (int k = 0; k < PK_EACH; ++k)
            if (k >= valid) m[k] = r[k] = 0.f;               // (what lies behind the end: codes of zero scales, no numbers)
        }
        uint32_t random[PK_EACH], w[2];
        if constexpr (RANDOM) {
          const uint32_t from = f.key + (uint32_t)at + (uint32_t)((uint64_t)at >> 32) * 0x9e3779b1u;
#pragma unroll
          for (int k = 0; k < PK_EACH; ++k) random[k] = aw_mix(from + (uint32_t)k);
        }
        const uint32_t Em = aw_encode<3, RANDOM>(m, random, w);
        aw_store_codes(t.m, at, valid, w);
        const uint32_t Ev = aw_encode<4, RANDOM>(r, random, w);
        aw_store_codes(t.v, at, valid, w);
        if (valid > 0 && threadIdx.x % AW_LANES == 0) {
          t.scale[at / AW_GROUP] = (uint8_t)Em;
          t.scale[groups + at / AW_GROUP] = (uint8_t)Ev;
        }
      } else {
        pk_row<float>::store(static_cast<float *>(t.m) + at, valid, m);
        pk_row<float>::store(static_cast<float *>(t.v) + at, valid, v);
      }
    }
  }
  // All blocks have read the counts when the last one arrives: it counts them up.
  __syncthreads();
  if (threadIdx.x >= HC_WAVE) return;
  unsigned *arrived = reinterpret_cast<unsigned *>(a.t[0].step + 1);
  int last = 0;
  if (threadIdx.x == 0) last = atomicAdd(arrived, 1u) == gridDim.x - 1u ? 1 : 0;
  if (__builtin_amdgcn_readfirstlane(last) == 0) return;
  if ((int)threadIdx.x < a.count) a.t[threadIdx.x].step[0] += 1;
  if (threadIdx.x == 0) atomicExch(arrived, 0u);
}

struct AwRead {
  const void *m[AW_MAX], *v[AW_MAX];
  const uint8_t *scale[AW_MAX];
  void *to_m[AW_MAX], *to_v[AW_MAX];
  int64_t n[AW_MAX];
  uint32_t first[AW_MAX + 1];
  int count;
};

// What states of 8 bits stand for: m and r.
template <typename T>
__global__ __launch_bounds__(HC_BLOCK) void aw_read(AwRead a) {
  uint32_t piece = blockIdx.x;
  const uint32_t pieces = a.first[a.count];
  for (int i = 0; piece < pieces; piece += gridDim.x) {
    while (piece >= a.first[i + 1]) ++i;
    const int64_t n = a.n[i], groups = (n + AW_GROUP - 1) / AW_GROUP;
    const int64_t at = (int64_t)(piece - a.first[i]) * AW_PIECE + (int64_t)threadIdx.x * PK_EACH;
    const int64_t left = n - at;
    if (left <= 0) continue;
    const int valid = left >= PK_EACH ? PK_EACH : (int)left;
    uint32_t w[2];
    float v[PK_EACH];
    aw_load_codes(a.m[i], at, valid, w);
    const uint32_t Em = a.scale[i][at / AW_GROUP], Ev = a.scale[i][groups + at / AW_GROUP];
    aw_decode<3>(w, Em, v);
#pragma unroll
    for (int k = 0; k < PK_EACH; ++k) v[k] += aw_poison(Em);
    pk_row<T>::store(static_cast<T *>(a.to_m[i]) + at, valid, v);
    aw_load_codes(a.v[i], at, valid, w);
    aw_decode<4>(w, Ev, v);
#pragma unroll
    for (int k = 0; k < PK_EACH; ++k) v[k] += aw_poison(Ev);
    pk_row<T>::store(static_cast<T *>(a.to_v[i]) + at, valid, v);
  }
}

// Pieces of tensors from..., at most AW_MAX of them and as many as a launch can number; how many there are.
static int aw_pieces(const int64_t *numel, int count, uint32_t *first) {
  uint64_t pieces = 0;
  int k = 0;
  for (; k < count && k < AW_MAX; ++k) {
    first[k] = (uint32_t)pieces;
    pieces += (uint64_t)((numel[k] + AW_PIECE - 1) / AW_PIECE);
    if (pieces > 0x7fffffffull) return k;
  }
  first[k] = (uint32_t)pieces;
  return k;
}

static dim3 aw_grid(uint32_t pieces) { return dim3(pieces < 1 ? 1 : pieces < AW_BLOCKS ? pieces : AW_BLOCKS); }

}  // namespace

extern "C" int hc_adamw_step(int count, void *const *param, const void *const *grad, int dtype, void *const *exp_avg,
                             void *const *exp_avg_sq, uint8_t *const *scale, float *const *master, int64_t *const *step,
                             const int64_t *numel, int state_bits, double lr, const float *lr_dev, double beta1, double beta2,
                             double eps, double weight_decay, void *stream) {
  const bool random = state_bits == (8 | HC_ADAMW_RANDOM);
  if (random) state_bits = 8;
  HC_REQUIRE(count >= 0 && (state_bits == 8 || state_bits == 32));
  HC_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0);
  if (dtype < HC_F32 || dtype > HC_BF16) return HC_EDTYPE;
  if (count == 0) return HC_OK;
  HC_REQUIRE(param && grad && exp_avg && exp_avg_sq && step && numel && (state_bits == 32) == (scale == nullptr));
  HC_REQUIRE(master == nullptr || dtype != HC_F32);
  for (int k = 0; k < count; ++k) {
    HC_REQUIRE(numel[k] >= 0 && step[k]);
    HC_REQUIRE(numel[k] == 0 || (param[k] && grad[k] && exp_avg[k] && exp_avg_sq[k] && (!scale || scale[k]) &&
                                 (!master || master[k])));
    if (numel[k] > (int64_t)0x7fffffff * AW_PIECE) return HC_EUNSUPPORTED;
  }
  AwArgs a;
  a.lr = lr;
  a.b1 = beta1;
  a.b2 = beta2;
  a.decay = weight_decay;
  a.lr_dev = lr_dev;
  a.eps = (float)eps;
  for (int from = 0; from < count; from += a.count) {
    a.count = aw_pieces(numel + from, count - from, a.first);
    for (int k = 0; k < a.count; ++k)
      a.t[k] = AwTensor{param[from + k],   grad[from + k],          exp_avg[from + k], exp_avg_sq[from + k],
                        scale ? scale[from + k] : nullptr, master ? master[from + k] : nullptr, step[from + k], numel[from + k]};
    const dim3 grid = aw_grid(a.first[a.count]), block(HC_BLOCK);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const auto launch = [&](auto type) {
      typedef decltype(type) T;
      const auto with_copy = [&](auto copy) {
        constexpr bool MASTER = decltype(copy)::value;
        if (state_bits == 32) aw_step<T, 32, MASTER, false><<<grid, block, 0, st>>>(a);
        else if (random) aw_step<T, 8, MASTER, true><<<grid, block, 0, st>>>(a);
        else aw_step<T, 8, MASTER, false><<<grid, block, 0, st>>>(a);
      };
      if constexpr (!std::is_same<T, float>::value) {
        if (master) return with_copy(std::true_type{});
      }
      with_copy(std::false_type{});
    };
    if (dtype == HC_F32) launch(float{});
    else if (dtype == HC_F16) launch(__half{});
    else launch(__hip_bfloat16{});
    if (const int rc = hc_launch_status()) return rc;
  }
  return HC_OK;
}

extern "C" int hc_adamw_moments(int count, const void *const *exp_avg, const void *const *exp_avg_sq,
                                const uint8_t *const *scale, const int64_t *numel, void *const *to_avg, void *const *to_root,
                                int dtype, void *stream) {
  HC_REQUIRE(count >= 0);
  if (dtype < HC_F32 || dtype > HC_BF16) return HC_EDTYPE;
  if (count == 0) return HC_OK;
  HC_REQUIRE(exp_avg && exp_avg_sq && scale && numel && to_avg && to_root);
  for (int k = 0; k < count; ++k) {
    HC_REQUIRE(numel[k] >= 0 && (numel[k] == 0 || (exp_avg[k] && exp_avg_sq[k] && scale[k] && to_avg[k] && to_root[k])));
    if (numel[k] > (int64_t)0x7fffffff * AW_PIECE) return HC_EUNSUPPORTED;
  }
  AwRead a;
  for (int from = 0; from < count; from += a.count) {
    a.count = aw_pieces(numel + from, count - from, a.first);
    for (int k = 0; k < a.count; ++k) {
      a.m[k] = exp_avg[from + k];
      a.v[k] = exp_avg_sq[from + k];
      a.scale[k] = scale[from + k];
      a.to_m[k] = to_avg[from + k];
      a.to_v[k] = to_root[from + k];
      a.n[k] = numel[from + k];
    }
    const dim3 grid = aw_grid(a.first[a.count]), block(HC_BLOCK);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == HC_F32) aw_read<float><<<grid, block, 0, st>>>(a);
    else if (dtype == HC_F16) aw_read<__half><<<grid, block, 0, st>>>(a);
    else aw_read<__hip_bfloat16><<<grid, block, 0, st>>>(a);
    if (const int rc = hc_launch_status()) return rc;
  }
  return HC_OK;
}
