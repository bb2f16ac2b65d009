// Rows sorted by expert and back.  A row i names top_k experts; pair q = i * top_k + j is its j-th choice.
//
// hc_expert_order: stable counting sort of the pairs by expert.  offset[e] is the first place of expert e; pair[place] = q
// and slot[q] = place for the pairs that name an expert, -1 for the others (whose places lie behind offset[E]).
//   One block sorts up to OR_SMALL_PAIRS pairs in one launch.  More take three: every block counts its chunk of pairs by
//   expert, a block per expert turns the counts of the chunks into first places, every block places its chunk.  Inside a
//   chunk a wave owns a run of adjacent pairs and takes 64 at a time: lanes with the same expert find each other by
//   ballots over the bits of the expert's number, so that places ascend with the pair whatever the scheduling.
//   Bound by its launches: 65 644 pairs of 64 experts 5 + 3 + 6 us, 400 006 of 8 5 + 6 + 7 (the middle one walks an expert's chunks
//   64 at a time, each behind the one before), eight pairs 2.6.
//
// hc_rows_to_experts: rows[place] = x[pair[place] / top_k], zeros behind offset[E].  Walks the rows of x, each read once
//   and stored at its top_k places.
// hc_rows_from_experts: out[i] = sum_j weight[q] * y[slot[q]] in the order of j, summed in fp32 (weight NULL: 1, which is
//   the gradient of hc_rows_to_experts).
// hc_rows_from_experts_grad: grad_y[place] = weight[q] * g[i], zeros behind offset[E], and grad_weight[q] = <g[i], y[slot[q]]>.
// All are bound by the rows' way through memory (a plain copy reaches 4.7 TB/s, a fill 6.8).  In a training pass (one kernel after
// the other, each with its own matrices) 16 411 rows of 1 024 bf16 to four experts / back with weights / the gradient of that / of
// the way there: 30 / 48 / 58 / 34 us, 5.7 / 3.4 / 5.2 / 4.9 TB/s; 200 003 rows of 256 fp32 to two: 111 / 125 / 178 / 91, 5.5 / 4.6 /
// 5.5 / 6.3.  A row's choices are read side by side (one after the other: 195 us for all of the first case, 181 so).
#include "hc_common.h"

namespace {

constexpr int OR_MAX_EXPERTS = 1024;
constexpr int OR_SMALL_PAIRS = 8192;
constexpr int OR_SMALL_BLOCK = 1024;
constexpr int OR_ROUNDS = 4;              // pairs of a lane that are held in registers
constexpr int OR_RUN = OR_ROUNDS * HC_WAVE;
constexpr int OR_CHUNK = OR_RUN * HC_WAVES_PER_BLOCK;
constexpr int OR_MAX_CHUNKS = 4096;

// The expert of a pair, E ("nowhere") for any number outside [0, E).
__device__ __forceinline__ int or_expert(const int64_t *__restrict__ expert, int64_t q, int E) {
  const int64_t e = expert[q];
  return e >= 0 && e < E ? (int)e : E;
}

// Places 64 pairs, one a lane (`on`: there is one): `next` (LDS, E + 1 counters of this wave) holds the next place of each
// expert.  Lanes with the same expert find each other by ballots over the bits of its number; the first of them moves the counter.
__device__ __forceinline__ void or_place(int64_t q, bool on, int e, int E, int bits, int *next, int32_t *__restrict__ slot,
                                         int32_t *__restrict__ pair) {
  const int lane = hc_lane();
  uint64_t same = __ballot(on);
  for (int b = 0; b < bits; ++b) {
    const uint64_t set = __ballot((e >> b) & 1);
    same &= (e >> b) & 1 ? set : ~set;
  }
  const int rank = __popcll(same & ((1ull << lane) - 1ull)), first = on ? __ffsll((long long)same) - 1 : lane;
  int place = 0;
  if (on && first == lane) place = atomicAdd(&next[e], __popcll(same));
  place = __shfl(place, first, HC_WAVE) + rank;
  if (on) {
    slot[q] = e < E ? place : -1;
    pair[place] = e < E ? (int32_t)q : -1;
  }
}

// Exclusive prefix sums of cnt[0 .. m) in LDS by one wave; returns the total.
__device__ __forceinline__ int or_scan(int *cnt, int m) {
  const int lane = hc_lane();
  int before = 0;
  for (int i0 = 0; i0 < m; i0 += HC_WAVE) {
    const int v = i0 + lane < m ? cnt[i0 + lane] : 0;
    int s = v;
#pragma unroll
    for (int d = 1; d < HC_WAVE; d *= 2) {
      const int o = __shfl_up(s, d, HC_WAVE);
      if (lane >= d) s += o;
    }
    if (i0 + lane < m) cnt[i0 + lane] = before + s - v;
    before += __shfl(s, HC_WAVE - 1, HC_WAVE);
  }
  return before;
}

// A wave's run of ROUNDS * 64 adjacent pairs from `lo` on: their experts (0 behind `hi`, where no pair is).
template <int ROUNDS>
__device__ __forceinline__ void or_load(const int64_t *__restrict__ expert, int64_t lo, int64_t hi, int E, int (&e)[ROUNDS]) {
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int64_t q = lo + r * HC_WAVE + hc_lane();
    e[r] = q < hi ? or_expert(expert, q, E) : 0;
  }
}

// Everything in one block of 64 pairs a wave and round: a row of E + 1 counters for each wave, one for the sums (69 700 bytes of LDS
// with sixteen waves and 1 024 experts, of the 160 KB that a launch may ask for on this device).
template <int ROUNDS>
__global__ __launch_bounds__(OR_SMALL_BLOCK) void or_small(const int64_t *__restrict__ expert, int32_t *__restrict__ slot,
                                                            int32_t *__restrict__ pair, int64_t *__restrict__ offset, int P,
                                                            int E, int bits) {
  extern __shared__ int s_cnt[];
  const int waves = (int)(blockDim.x / HC_WAVE), wave = hc_wave_in_block(), lane = hc_lane(), bins = E + 1;
  int *sum = s_cnt + waves * bins, *mine = s_cnt + wave * bins, e[ROUNDS];
  const int lo = wave * ROUNDS * HC_WAVE;
  or_load<ROUNDS>(expert, lo, P, E, e);
  for (int i = (int)threadIdx.x; i < (waves + 1) * bins; i += (int)blockDim.x) s_cnt[i] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if (lo + r * HC_WAVE + lane < P) atomicAdd(&mine[e[r]], 1);
  __syncthreads();
  for (int b = (int)threadIdx.x; b < bins; b += (int)blockDim.x) {
    int s = 0;
    for (int w = 0; w < waves; ++w) {
      const int c = s_cnt[w * bins + b];
      s_cnt[w * bins + b] = s;
      s += c;
    }
    sum[b] = s;
  }
  __syncthreads();
  if (wave == 0) or_scan(sum, bins);
  __syncthreads();
  for (int b = (int)threadIdx.x; b < bins; b += (int)blockDim.x) {
    offset[b] = sum[b];
    for (int w = 0; w < waves; ++w) s_cnt[w * bins + b] += sum[b];
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if (lo + r * HC_WAVE < P) or_place(lo + r * HC_WAVE + lane, lo + r * HC_WAVE + lane < P, e[r], E, bits, mine, slot, pair);
}

__global__ __launch_bounds__(HC_BLOCK) void or_count(const int64_t *__restrict__ expert, int *__restrict__ count, int64_t P,
                                                     int E, int64_t chunk) {
  extern __shared__ int s_cnt[];
  const int bins = E + 1;
  for (int e = (int)threadIdx.x; e < bins; e += HC_BLOCK) s_cnt[e] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * chunk, hi = lo + chunk < P ? lo + chunk : P;
  for (int64_t q0 = lo + hc_wave_in_block() * OR_RUN; q0 < hi; q0 += OR_CHUNK) {
    int e[OR_ROUNDS];
    or_load<OR_ROUNDS>(expert, q0, hi, E, e);
#pragma unroll
    for (int r = 0; r < OR_ROUNDS; ++r)
      if (q0 + r * HC_WAVE + hc_lane() < hi) atomicAdd(&s_cnt[e[r]], 1);
  }
  __syncthreads();
  for (int e = (int)threadIdx.x; e < bins; e += HC_BLOCK) count[(int64_t)e * gridDim.x + blockIdx.x] = s_cnt[e];
}

// count[e][chunk] becomes the number of e's pairs in the chunks before; total[e] their number in all.
__global__ __launch_bounds__(HC_WAVE) void or_prefix(int *__restrict__ count, int *__restrict__ total, int chunks) {
  int *row = count + (int64_t)blockIdx.x * chunks;
  const int t = or_scan(row, chunks);
  if (hc_lane() == 0) total[blockIdx.x] = t;
}

// The chunk's pairs in pieces of OR_CHUNK, a run of each by every wave.
__global__ __launch_bounds__(HC_BLOCK) void or_scatter(const int64_t *__restrict__ expert, const int *__restrict__ count,
                                                       const int *__restrict__ total, int32_t *__restrict__ slot,
                                                       int32_t *__restrict__ pair, int64_t *__restrict__ offset, int64_t P,
                                                       int E, int64_t chunk, int bits) {
  extern __shared__ int s_cnt[];
  constexpr int W = HC_WAVES_PER_BLOCK;
  const int wave = hc_wave_in_block(), lane = hc_lane(), bins = E + 1;
  int *sum = s_cnt + W * bins, *mine = s_cnt + wave * bins, e[OR_ROUNDS];
  const int64_t lo = (int64_t)blockIdx.x * chunk, hi = lo + chunk < P ? lo + chunk : P;
  or_load<OR_ROUNDS>(expert, lo + wave * OR_RUN, hi, E, e);
  for (int b = (int)threadIdx.x; b < bins; b += HC_BLOCK) sum[b] = total[b];
  __syncthreads();
  if (wave == 0) or_scan(sum, bins);
  __syncthreads();
  for (int b = (int)threadIdx.x; b < bins; b += HC_BLOCK) {
    if (blockIdx.x == 0) offset[b] = sum[b];
    sum[b] += count[(int64_t)b * gridDim.x + blockIdx.x];
  }
  for (int64_t piece = lo; piece < hi; piece += OR_CHUNK) {
    const int64_t q0 = piece + wave * OR_RUN;
    if (piece > lo) or_load<OR_ROUNDS>(expert, q0, hi, E, e);
    for (int i = (int)threadIdx.x; i < W * bins; i += HC_BLOCK) s_cnt[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < OR_ROUNDS; ++r)
      if (q0 + r * HC_WAVE + lane < hi) atomicAdd(&mine[e[r]], 1);
    __syncthreads();
    for (int b = (int)threadIdx.x; b < bins; b += HC_BLOCK) {
      int s = sum[b];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int c = s_cnt[w * bins + b];
        s_cnt[w * bins + b] = s;
        s += c;
      }
      sum[b] = s;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < OR_ROUNDS; ++r)
      if (q0 + r * HC_WAVE < hi) or_place(q0 + r * HC_WAVE + lane, q0 + r * HC_WAVE + lane < hi, e[r], E, bits, mine, slot, pair);
    __syncthreads();
  }
}

struct OrShape {
  int64_t chunk, chunks;
};

static OrShape or_shape(int64_t P) {
  OrShape s;
  s.chunk = OR_CHUNK;
  while ((P + s.chunk - 1) / s.chunk > OR_MAX_CHUNKS) s.chunk *= 2;
  s.chunks = (P + s.chunk - 1) / s.chunk;
  return s;
}

// ---- rows ------------------------------------------------------------------
// A row is D elements in pieces of VEC; a thread owns one piece of one row.  ANY: pieces of 16 bytes at the alignment of one
// element, the last one moved back to the row's end: what it shares with the one before it is computed and stored by both, with
// the same bits.  Else rows are whole pieces at their own alignment.  (To two experts / back, us, by the pieces that the
// alignment allows and by ANY: 100 000 rows of 602 bf16 115 / 137 and 71 / 65; 200 000 of 601 379 / 480 and 150 / 134; 100 000 of 602
// fp32 139 / 206 and 153 / 129.)
typedef uint32_t mv_words_2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t mv_words_4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T, int VEC, bool ANY>
struct mv_row {
  typedef typename std::conditional<sizeof(T) == 2, mv_words_2, mv_words_4>::type any_t;
  typedef typename std::conditional<ANY, any_t, typename hc_vec<T, VEC>::raw_t>::type raw;
  union U {
    raw whole;
    T e[VEC];
    __device__ U() {}
  };
  __device__ __forceinline__ static int column(int piece, int D) {
    const int c = piece * VEC;
    return ANY && c > D - VEC ? D - VEC : c;
  }
  __device__ __forceinline__ static raw get(const T *p) { return *reinterpret_cast<const raw *>(p); }
  __device__ __forceinline__ static void set(T *p, raw v) { *reinterpret_cast<raw *>(p) = v; }
  template <bool NT = false>
  __device__ __forceinline__ static void load(const T *p, float (&out)[VEC]) {
    if constexpr (NT && !ANY) {
      hc_vec<T, VEC>::load_nt(p, out);
    } else {
      U u;
      if constexpr (NT) u.whole = __builtin_nontemporal_load(reinterpret_cast<const raw *>(p));
      else u.whole = get(p);
#pragma unroll
      for (int i = 0; i < VEC; ++i) out[i] = hc_to_f32<T>(u.e[i]);
    }
  }
  __device__ __forceinline__ static void store(T *p, const float (&in)[VEC]) {
    U u;
#pragma unroll
    for (int i = 0; i < VEC; ++i) u.e[i] = hc_from_f32<T>(in[i]);
    set(p, u.whole);
  }
};

struct MvArgs {
  int64_t n, P;
  int D, k, pieces, E;
  const int32_t *slot;
  const int64_t *offset;
};

// The place of a pair, -1 if it has none (or one that is not among the P).
__device__ __forceinline__ int32_t mv_slot(const MvArgs &a, int64_t q) {
  const int32_t s = a.slot[q];
  return s < a.P ? s : -1;
}

template <typename T, int VEC, bool ANY>
__device__ __forceinline__ void mv_zero_tail(const MvArgs &a, T *__restrict__ rows) {
  typedef mv_row<T, VEC, ANY> row;
  const int64_t end = a.offset[a.E], live = end < 0 ? 0 : end, rest = (a.P - live) * a.pieces;
  for (int64_t i = (int64_t)blockIdx.x * HC_BLOCK + threadIdx.x; i < rest; i += (int64_t)gridDim.x * HC_BLOCK)
    row::set(rows + (live + i / a.pieces) * a.D + row::column((int)(i % a.pieces), a.D), typename row::raw{});
}

template <typename T, int VEC, bool ANY>
__global__ __launch_bounds__(HC_BLOCK) void mv_to(MvArgs a, const T *__restrict__ x, T *__restrict__ rows) {
  typedef mv_row<T, VEC, ANY> row;
  const uint32_t item = blockIdx.x * HC_BLOCK + threadIdx.x;       // (a launch has less than 2^32 threads)
  const int64_t i = item / (uint32_t)a.pieces;
  if (i < a.n) {
    const int c = row::column((int)(item - (uint32_t)i * (uint32_t)a.pieces), a.D);
    const typename row::raw v = row::get(x + i * a.D + c);
    for (int j = 0; j < a.k; ++j) {
      const int32_t s = mv_slot(a, i * a.k + j);
      if (s >= 0) row::set(rows + (int64_t)s * a.D + c, v);
    }
  }
  mv_zero_tail<T, VEC, ANY>(a, rows);
}

// K: the choices of a row that are read at a time.
template <typename T, int VEC, bool ANY, int K>
__global__ __launch_bounds__(HC_BLOCK) void mv_from(MvArgs a, const T *__restrict__ y, const float *__restrict__ weight,
                                                    T *__restrict__ out) {
  typedef mv_row<T, VEC, ANY> row;
  const uint32_t item = blockIdx.x * HC_BLOCK + threadIdx.x;       // (a launch has less than 2^32 threads)
  const int64_t i = item / (uint32_t)a.pieces;
  if (i >= a.n) return;
  const int c = row::column((int)(item - (uint32_t)i * (uint32_t)a.pieces), a.D);
  float sum[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) sum[v] = 0.f;
  for (int j0 = 0; j0 < a.k; j0 += K) {
    int32_t s[K];
    float w[K], p[K][VEC];
#pragma unroll
    for (int j = 0; j < K; ++j) s[j] = j0 + j < a.k ? mv_slot(a, i * a.k + j0 + j) : -1;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      w[j] = weight != nullptr && s[j] >= 0 ? weight[i * a.k + j0 + j] : 1.f;
      if (s[j] >= 0 && weight != nullptr) {
        row::load(y + (int64_t)s[j] * a.D + c, p[j]);
      } else if (s[j] >= 0) {
        // gradients: nothing reads them after this.  (In the passes above, plain / non-temporal: 43 / 34 and 101 / 91 us; what the last-level
        // cache then holds makes the next pass's sum with weights take 42 / 48 and 116 / 125: both together 85 / 82 and 217 / 216.)
        row::template load<true>(y + (int64_t)s[j] * a.D + c, p[j]);
      } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v) p[j][v] = 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int v = 0; v < VEC; ++v) sum[v] = fmaf(w[j], p[j][v], sum[v]);
  }
  row::store(out + i * a.D + c, sum);
}

// L lanes a row; K as above.
template <typename T, int VEC, bool ANY, int K>
__global__ __launch_bounds__(HC_BLOCK) void mv_from_grad(MvArgs a, const T *__restrict__ g, const T *__restrict__ y,
                                                         const float *__restrict__ weight, T *__restrict__ grad_y,
                                                         float *__restrict__ grad_weight, int L) {
  typedef mv_row<T, VEC, ANY> row;
  const int lane = (int)threadIdx.x & (L - 1);
  const int64_t i = ((int64_t)blockIdx.x * HC_BLOCK + threadIdx.x) / L;
  if (i < a.n) {
    for (int j0 = 0; j0 < a.k; j0 += K) {
      int32_t s[K];
      float w[K], dot[K];
#pragma unroll
      for (int j = 0; j < K; ++j) {
        s[j] = j0 + j < a.k ? mv_slot(a, i * a.k + j0 + j) : -1;
        w[j] = s[j] >= 0 ? weight[i * a.k + j0 + j] : 0.f;
        dot[j] = 0.f;
      }
      for (int p = lane; p < a.pieces; p += L) {
        float gv[VEC], yv[K][VEC];
        const int c = row::column(p, a.D), twice = p * VEC - c;         // elements that the piece before has counted
        row::load(g + i * a.D + c, gv);
#pragma unroll
        for (int j = 0; j < K; ++j)
          if (s[j] >= 0) row::load(y + (int64_t)s[j] * a.D + c, yv[j]);
#pragma unroll
        for (int j = 0; j < K; ++j)
          if (s[j] >= 0) {
            float o[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
              dot[j] = !ANY || v >= twice ? fmaf(gv[v], yv[j][v], dot[j]) : dot[j];
              o[v] = w[j] * gv[v];
            }
            row::store(grad_y + (int64_t)s[j] * a.D + c, o);
          }
      }
#pragma unroll
      for (int j = 0; j < K; ++j) {
        for (int d = L / 2; d >= 1; d /= 2) dot[j] += __shfl_xor(dot[j], d, HC_WAVE);
        if (lane == 0 && j0 + j < a.k) grad_weight[i * a.k + j0 + j] = dot[j];
      }
    }
  }
  mv_zero_tail<T, VEC, ANY>(a, grad_y);
}

// As many choices at a time as a row has, up to four.
template <typename F>
static int mv_with_choices(int64_t k, F &&f) {
  if (k == 1) return f(std::integral_constant<int, 1>{});
  if (k == 2) return f(std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, 4>{});
}

static bool mv_args(int64_t n, int64_t top_k, int64_t E, int64_t D, const int32_t *slot, const int64_t *offset, MvArgs *a) {
  if (n < 0 || top_k < 1 || E < 1 || D < 1) return false;
  a->n = n;
  a->P = (int64_t)((uint64_t)n * (uint64_t)top_k);          // (below 2^31, or the call is refused)
  a->D = (int)D;
  a->k = (int)top_k;
  a->E = (int)E;
  a->slot = slot;
  a->offset = offset;
  return true;
}

// Fewer than 2^31 pairs, as hc_expert_order sorts.
static bool mv_sizes_ok(int64_t n, int64_t top_k, int64_t E, int64_t D) {
  return D < (1 << 30) && n <= ((1ll << 31) - 1) / top_k && top_k < (1ll << 31) && E <= OR_MAX_EXPERTS;
}

// Elements of T in a piece, and whether it may lie at any element: 16 bytes, for rows that are shorter as many as their length and
// the matrices' alignment allow.
template <typename T, typename F>
static int mv_with_piece(uintptr_t at, int64_t D, F &&f) {
  constexpr int MOST = 16 / (int)sizeof(T);
  const uint64_t a = (uint64_t)at | (uint64_t)D * sizeof(T);
  if (a % 16 == 0) return f(std::integral_constant<int, MOST>{}, std::false_type{});
  if (D >= MOST) return f(std::integral_constant<int, MOST>{}, std::true_type{});
  if (a % 8 == 0) return f(std::integral_constant<int, 8 / (int)sizeof(T)>{}, std::false_type{});
  if (a % 4 == 0) return f(std::integral_constant<int, 4 / (int)sizeof(T)>{}, std::false_type{});
  return f(std::integral_constant<int, 1>{}, std::false_type{});
}

template <typename F>
static int mv_with_type(int dtype, F &&f) {
  if (dtype == HC_F32) return f(float{});
  if (dtype == HC_F16) return f(__half{});
  if (dtype == HC_BF16) return f(__hip_bfloat16{});
  return HC_EDTYPE;
}

static bool or_sizes_ok(int64_t pairs, int64_t E) { return pairs < (1ll << 31) && E <= OR_MAX_EXPERTS; }

}  // namespace

extern "C" size_t hc_expert_order_workspace_bytes(int64_t pairs, int64_t E) {
  if (pairs < 0 || E < 1 || !or_sizes_ok(pairs, E) || pairs <= OR_SMALL_PAIRS) return 0;
  return hc_align_up((size_t)(E + 1) * (size_t)(or_shape(pairs).chunks + 1) * sizeof(int), 256);
}

extern "C" int hc_expert_order(const int64_t *expert, int64_t pairs, int64_t E, int32_t *slot, int32_t *pair,
                               int64_t *offset, void *workspace, size_t workspace_bytes, void *stream) {
  HC_REQUIRE(pairs >= 0 && E >= 1);
  if (!or_sizes_ok(pairs, E)) return HC_EUNSUPPORTED;
  HC_REQUIRE(offset && (pairs == 0 || (expert && slot && pair)));
  hipStream_t st = static_cast<hipStream_t>(stream);
  int bits = 1;
  while ((1 << bits) < E + 1) ++bits;
  const size_t bins = (size_t)E + 1;
  if (pairs <= OR_SMALL_PAIRS) {
    // as many waves as sixteen rounds of two or eight need
    const int rounds = pairs <= 2 * OR_SMALL_BLOCK ? 2 : OR_SMALL_PAIRS / OR_SMALL_BLOCK;
    int waves = (int)((pairs + rounds * HC_WAVE - 1) / (rounds * HC_WAVE));
    waves = waves < 1 ? 1 : waves;
    const auto kernel = rounds == 2 ? or_small<2> : or_small<OR_SMALL_PAIRS / OR_SMALL_BLOCK>;
    kernel<<<dim3(1), dim3((unsigned)waves * HC_WAVE), (waves + 1) * bins * sizeof(int), st>>>(expert, slot, pair, offset, (int)pairs,
                                                                                              (int)E, bits);
    return hc_launch_status();
  }
  const OrShape s = or_shape(pairs);
  if (!workspace || workspace_bytes < hc_expert_order_workspace_bytes(pairs, E) || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return HC_EWORKSPACE;
  int *count = static_cast<int *>(workspace), *total = count + bins * s.chunks;
  or_count<<<dim3((unsigned)s.chunks), dim3(HC_BLOCK), bins * sizeof(int), st>>>(expert, count, pairs, (int)E, s.chunk);
  or_prefix<<<dim3((unsigned)bins), dim3(HC_WAVE), 0, st>>>(count, total, (int)s.chunks);
  or_scatter<<<dim3((unsigned)s.chunks), dim3(HC_BLOCK), (HC_WAVES_PER_BLOCK + 1) * bins * sizeof(int), st>>>(
      expert, count, total, slot, pair, offset, pairs, (int)E, s.chunk, bits);
  return hc_launch_status();
}

extern "C" int hc_rows_to_experts(const void *x, int dtype, int64_t n, int64_t top_k, int64_t E, int64_t D,
                                  const int32_t *slot, const int64_t *offset, void *rows, void *stream) {
  MvArgs a;
  HC_REQUIRE(mv_args(n, top_k, E, D, slot, offset, &a));
  if (!mv_sizes_ok(n, top_k, E, D)) return HC_EUNSUPPORTED;
  if (n == 0) return dtype >= HC_F32 && dtype <= HC_BF16 ? HC_OK : HC_EDTYPE;
  HC_REQUIRE(x && slot && offset && rows);
  return mv_with_type(dtype, [&](auto type) {
    typedef decltype(type) T;
    return mv_with_piece<T>(reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(rows), D, [&](auto piece, auto any) {
      constexpr int VEC = decltype(piece)::value;
      constexpr bool ANY = decltype(any)::value;
      a.pieces = (int)((D + VEC - 1) / VEC);
      const int64_t blocks = (n * a.pieces + HC_BLOCK - 1) / HC_BLOCK;
      if (!hc_grid_ok(blocks)) return (int)HC_EUNSUPPORTED;
      mv_to<T, VEC, ANY><<<dim3((unsigned)blocks), dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(
          a, static_cast<const T *>(x), static_cast<T *>(rows));
      return hc_launch_status();
    });
  });
}

extern "C" int hc_rows_from_experts(const void *y, int dtype, int64_t n, int64_t top_k, int64_t E, int64_t D,
                                    const int32_t *slot, const float *weight, void *out, void *stream) {
  MvArgs a;
  HC_REQUIRE(mv_args(n, top_k, E, D, slot, nullptr, &a));
  if (!mv_sizes_ok(n, top_k, E, D)) return HC_EUNSUPPORTED;
  if (n == 0) return dtype >= HC_F32 && dtype <= HC_BF16 ? HC_OK : HC_EDTYPE;
  HC_REQUIRE(y && slot && out);
  return mv_with_type(dtype, [&](auto type) {
    typedef decltype(type) T;
    return mv_with_piece<T>(reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(out), D, [&](auto piece, auto any) {
      constexpr int VEC = decltype(piece)::value;
      constexpr bool ANY = decltype(any)::value;
      a.pieces = (int)((D + VEC - 1) / VEC);
      const int64_t blocks = (n * a.pieces + HC_BLOCK - 1) / HC_BLOCK;
      if (!hc_grid_ok(blocks)) return (int)HC_EUNSUPPORTED;
      return mv_with_choices(top_k, [&](auto choices) {
        mv_from<T, VEC, ANY, decltype(choices)::value><<<dim3((unsigned)blocks), dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(
            a, static_cast<const T *>(y), weight, static_cast<T *>(out));
        return hc_launch_status();
      });
    });
  });
}

extern "C" int hc_rows_from_experts_grad(const void *g, const void *y, int dtype, int64_t n, int64_t top_k, int64_t E,
                                         int64_t D, const int32_t *slot, const int64_t *offset, const float *weight,
                                         void *grad_y, float *grad_weight, void *stream) {
  MvArgs a;
  HC_REQUIRE(mv_args(n, top_k, E, D, slot, offset, &a));
  if (!mv_sizes_ok(n, top_k, E, D)) return HC_EUNSUPPORTED;
  if (n == 0) return dtype >= HC_F32 && dtype <= HC_BF16 ? HC_OK : HC_EDTYPE;
  HC_REQUIRE(g && y && slot && offset && weight && grad_y && grad_weight);
  return mv_with_type(dtype, [&](auto type) {
    typedef decltype(type) T;
    const uintptr_t at = reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(grad_y);
    return mv_with_piece<T>(at, D, [&](auto piece, auto any) {
      constexpr int VEC = decltype(piece)::value;
      constexpr bool ANY = decltype(any)::value;
      a.pieces = (int)((D + VEC - 1) / VEC);
      int L = 1;
      while (L < HC_WAVE && L < a.pieces) L *= 2;
      const int64_t blocks = (n * L + HC_BLOCK - 1) / HC_BLOCK;
      if (!hc_grid_ok(blocks)) return (int)HC_EUNSUPPORTED;
      return mv_with_choices(top_k, [&](auto choices) {
        mv_from_grad<T, VEC, ANY, decltype(choices)::value>
            <<<dim3((unsigned)blocks), dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(
                a, static_cast<const T *>(g), static_cast<const T *>(y), weight, static_cast<T *>(grad_y), grad_weight, L);
        return hc_launch_status();
      });
    });
  });
}
