// A tile of an expert product on the matrix cores: the kernels behind hc_expert_linear and hc_expert_linear_grad, a template
// that expert_f32.hip, expert_f16.hip and expert_bf16.hip fill in for their type.
//
//   result[P, Q] = sum over the inner index of p[P, inner] * q[Q, inner]
//     forward            P: rows of the batch, Q: rows of w[e],    inner: columns of both
//     gradient of x      P: rows of the batch, Q: columns of w[e], inner: rows of w[e]           (KN)
//     gradient of w      P: columns of g,      Q: columns of x,    inner: rows of the batch      (GRAD)
//
// Sums are held in fp32 and rounded once, to the type of the result.  Large products are bound by the matrix pipes and by what
// their feeding leaves of them: a step of a large tile reads 192 KB from LDS and writes 64, at 128 bytes a cycle as long as its
// products take -- 8 192 x 8 192 x 8 192 bf16 910 / 896 / 877 us (forward, gradient of x, of w with its join; 1 209 to
// 1 254 TFLOP/s), 32 771 rows of 16 experts of 2 048 x 1 024 bf16 169 / 157 / 159 (812 to 875), 8 192 x 4 096 x 4 096 fp32 1 979 / 1 948 /
// 1 934 (139 to 142) --, few rows at many experts by reading the matrices (16 rows at 15 of 2 048 x 1 024 bf16 12 us, 63 MB).  These are
// launches of one kind back to back; the three of a training pass take 528 us there (each by itself, under a profiler, 201 / 206 / 192).
#pragma once

#include "expert_find.h"

namespace {

typedef float el_acc __attribute__((ext_vector_type(16)));
typedef float el_four __attribute__((ext_vector_type(4)));
typedef short el_eight __attribute__((ext_vector_type(8)));
typedef short el_quad __attribute__((ext_vector_type(4)));
typedef uint32_t el_piece __attribute__((ext_vector_type(4)));
typedef uint32_t el_words __attribute__((ext_vector_type(4), aligned(4)));      // 16 bytes that start on 4

constexpr uint32_t EL_NOWHERE = 0xffffff00u;    // behind every buffer, as are the bytes that follow it: reads as zero
#define EL_LDS __attribute__((address_space(3)))

// 16 bytes of the inner index for 32 rows by each half of the wave; both operands go by the same order, so that which of the
// instruction's inner indices a value takes does not matter.
template <typename T>
struct el_type {
  typedef el_eight frag;
  __device__ __forceinline__ static el_acc mfma(frag a, frag b, el_acc c) {
    if constexpr (std::is_same<T, __half>::value) {
      typedef _Float16 f16 __attribute__((ext_vector_type(8)));
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16, a), __builtin_bit_cast(f16, b), c, 0, 0, 0);
    } else {
      typedef __bf16 b16 __attribute__((ext_vector_type(8)));
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16, a), __builtin_bit_cast(b16, b), c, 0, 0, 0);
    }
  }
};
template <>
struct el_type<float> {
  typedef el_four frag;
  __device__ __forceinline__ static el_acc mfma(frag a, frag b, el_acc c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

// A piece of an operand in LDS: W rows (columns) of the result by 128 bytes of inner index, in chunks of 16 bytes.
//   TR = false: inner index along memory, [W][ROWB]
//   TR = true:  inner index outside, [ROWB / size][W].  16 bits: read by ds_read_b64_tr_b16, 4 rows x 16 columns by 16 lanes; fp32:
//               read by columns
// Chunk c of row r lies at c ^ turn(r), so that the lanes that are served at a time find their values in different banks.
// DIRECT: chunks go straight into LDS, for operands whose rows start on 4 bytes; a step that ends inside a row goes there by
// words.  Else (16 bits, an odd width or address) the five words that hold a chunk's eight elements pass through registers, in
// which they are moved into place; of the words only the tensor's first and last can hold two bytes that are not its own.
template <typename T, int W, int ROWB, bool TR, int THREADS, bool DIRECT>
struct el_operand {
  static constexpr int PER = 16 / (int)sizeof(T), INNER = ROWB / (int)sizeof(T);
  static constexpr int CHUNKS = W * ROWB / 16, EACH = CHUNKS / THREADS;
  static_assert(CHUNKS % THREADS == 0, "whole chunks per thread");
  uint32_t at[EACH];        // byte offset of this thread's chunks in the operand's first piece (not DIRECT: of their first words)
  int first[EACH];          // first inner index (TR = false) or column of each
  el_piece held[DIRECT ? 1 : EACH];
  uint32_t last[DIRECT ? 1 : EACH], shift[DIRECT ? 1 : EACH];           // the fifth words; bytes in front of the first element
  uint32_t stride;          // of the operand's rows in elements
  int wide;                 // rows (TR = false) or columns (TR = true) that exist from the tile's first on

  // what is added, bit by bit, to the numbers of a row's chunks (TR: of its 32 bytes, of its 128 bytes where T is fp32)
  __device__ __forceinline__ static int turn(int r) {
    // (a row of 64 columns has four such pieces and takes half of the banks, those of wider tiles have eight and take them all)
    if constexpr (TR) return sizeof(T) == 4 ? (r >> 2) & 1 : W == 64 ? r & 2 : (r & 3) * 2 + ((r >> 3) & 1);
    else return ROWB == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
  }
  __device__ __forceinline__ void init(int t, uint32_t stride_, int wide_, uint32_t skip) {
    stride = stride_;
    wide = wide_;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int q = i * THREADS + t;
      int r, c;
      if constexpr (!TR) {
        r = q / (ROWB / 16);
        c = q % (ROWB / 16) ^ turn(r);
      } else {
        r = q / (W / PER);
        c = q % (W / PER) ^ turn(r) * (sizeof(T) == 2 ? 2 : 8);
      }
      first[i] = c * PER;
      at[i] = ((uint32_t)r * stride + (uint32_t)first[i]) * (uint32_t)sizeof(T);
      if constexpr (!DIRECT) {
        shift[i] = (at[i] + skip) & 2;
        at[i] = (at[i] + skip) & ~3u;
      }
      if ((TR ? first[i] : r) >= wide) at[i] = EL_NOWHERE;
    }
  }
  // left: inner indices from the piece's first on.  Columns behind the last one may hold what lies there (they are not part of
  // the result), inner indices behind the last one are zeros.
  __device__ __forceinline__ void fetch(hc_buffer b, EL_LDS char *lds, int t, int wave, int left) {
    if constexpr (DIRECT) {
      if (TR || left >= INNER || left % PER == 0) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          const uint32_t o = TR || first[i] < left ? at[i] : EL_NOWHERE;
          __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (EL_LDS void *)(lds + (i * THREADS + wave * HC_WAVE) * 16), 16, o, 0, 0, 0);
        }
      } else {
#pragma unroll 4
        for (int i = 0; i < EACH * 4; ++i) {
          const int q = i * THREADS + t, r = q / (ROWB / 4), c = (q % (ROWB / 4) / 4) ^ turn(r);
          const int k = (c * 4 + q % 4) * (4 / (int)sizeof(T));
          const uint32_t o = r < wide && k < left ? ((uint32_t)r * stride + (uint32_t)k) * (uint32_t)sizeof(T) : EL_NOWHERE;
          __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (EL_LDS void *)(lds + (i * THREADS + wave * HC_WAVE) * 4), 4, o, 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const uint32_t o = (TR ? (i * THREADS + t) / (W / PER) : first[i]) < left ? at[i] : EL_NOWHERE;
        held[i] = __builtin_amdgcn_raw_buffer_load_b128(b, o, 0, 0);
        last[i] = __builtin_amdgcn_raw_buffer_load_b32(b, o + 16, 0, 0);
      }
    }
  }
  __device__ __forceinline__ void put(EL_LDS char *lds, int t, int left) const {
    if constexpr (!DIRECT)
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        el_piece v;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          v[x] = __builtin_amdgcn_alignbyte(x < 3 ? held[i][x < 3 ? x + 1 : 3] : last[i], held[i][x], shift[i]);
          if (!TR) v[x] &= left >= first[i] + 2 * x + 2 ? ~0u : left > first[i] + 2 * x ? 0xffffu : 0u;
        }
        *(EL_LDS el_piece *)(lds + (i * THREADS + t) * 16) = v;
      }
  }
  // The fragment of 32 rows (columns) from `from` on in the k-th quarter of the piece: lane l has row from + l % 32 and of the
  // quarter's 32 bytes of inner index the half l / 32.
  __device__ __forceinline__ static typename el_type<T>::frag read(const EL_LDS char *lds, int from, int k) {
    const int lane = hc_lane();
    if constexpr (!TR) {
      const int r = from + (lane & 31), c = k * 2 + (lane >> 5);
      return *(const EL_LDS typename el_type<T>::frag *)(lds + r * ROWB + ((c ^ turn(lane)) * 16));
    } else if constexpr (sizeof(T) == 2) {
      const int i = lane & 15, g = lane >> 4;
      const int r = k * 16 + (g >> 1) * 8 + (i >> 2), c = from / 16 + (g & 1);
      const EL_LDS char *p = lds + r * (W * 2) + (i & 3) * 8;
      const el_quad a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((EL_LDS el_quad *)(p + ((c ^ turn(r)) * 32)));
      const el_quad b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((EL_LDS el_quad *)(p + 4 * (W * 2) + ((c ^ turn(r)) * 32)));
      return el_eight{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    } else {
      const EL_LDS float *p = (const EL_LDS float *)lds + (k * 8 + (lane >> 5) * 4) * W + ((from + (lane & 31)) ^ (lane >> 5) * 32);
      return el_four{p[0], p[W], p[2 * W], p[3 * W]};
    }
  }
};

// One step: the piece in `from` is multiplied while a later one is on its way to `to`.  A function of its own for the sake of the
// two restricted pointers: they tell the compiler that what is on its way is not what is read, without which it waits for
// all of it in front of every transposing read.
template <typename OP_P, typename OP_Q, int TP, int TQ, int BYTES_P, int QUARTERS, typename T>
__device__ __forceinline__ void el_step(const EL_LDS char *__restrict__ from, EL_LDS char *__restrict__ to, OP_P &fp, OP_Q &fq,
                                        hc_buffer bp, hc_buffer bq, bool more, int left, int t, int wave, int wp, int wq,
                                        el_acc (&acc)[TP][TQ]) {
  typedef typename el_type<T>::frag frag;
  if (more) {
    fp.fetch(bp, to, t, wave, left);
    fq.fetch(bq, to + BYTES_P, t, wave, left);
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int k = 0; k < QUARTERS; ++k) {
    frag u[TP], v[TQ];
#pragma unroll
    for (int i = 0; i < TP; ++i) u[i] = OP_P::read(from, wp + i * 32, k);
#pragma unroll
    for (int j = 0; j < TQ; ++j) v[j] = OP_Q::read(from + BYTES_P, wq + j * 32, k);
#pragma unroll
    for (int i = 0; i < TP; ++i)
#pragma unroll
      for (int j = 0; j < TQ; ++j) acc[i][j] = el_type<T>::mfma(v[j], u[i], acc[i][j]);
  }
}

// A block of WP x WQ waves computes BP x BQ of the result; its operands come in pieces of ROWB bytes of inner index through two
// stages in LDS, the next piece on its way while one is multiplied.  (Half pieces through five chunks of LDS, on their way up to
// two and a half pieces ahead and waited for by their number: 8 192 x 8 192 x 8 192 bf16 941 us where this took 976, but 100 000 x
// 256 x 256 30 where it took 27.)
template <typename T, int BP, int BQ, int WP, int WQ, int ROWB, bool GRAD, bool KN, bool DIRECT>
__global__ __launch_bounds__(WP *WQ *HC_WAVE, 2) void el_tile(ElProduct a) {
  constexpr int THREADS = WP * WQ * HC_WAVE, TP = BP / WP / 32, TQ = BQ / WQ / 32, PER = 16 / (int)sizeof(T);
  constexpr bool PT = GRAD, QT = GRAD || KN;
  typedef el_operand<T, BP, ROWB, PT, THREADS, DIRECT> op_p;
  typedef el_operand<T, BQ, ROWB, QT, THREADS, DIRECT> op_q;
  constexpr int BK = op_p::INNER, BYTES_P = BP * ROWB, STAGE = (BP + BQ) * ROWB;
  constexpr uint32_t SIZE = sizeof(T);
  constexpr int OUT = WP * WQ * 32 * (TQ * 32 + PER) * (int)sizeof(T), MEM = 2 * STAGE > OUT ? 2 * STAGE : OUT;
  __shared__ __attribute__((aligned(16))) char s_mem[MEM];
  EL_LDS char *lds = (EL_LDS char *)s_mem;
  const int64_t b = hc_xcd_block<!GRAD ? 8 : sizeof(T) == 2 ? 16 : 4>(blockIdx.x, gridDim.x);
  const int t = (int)threadIdx.x, lane = hc_lane(), wave = hc_wave_in_block();
  const int wp = wave % WP * (BP / WP), wq = wave / WP * (BQ / WQ);
  const uint32_t per = (uint32_t)(GRAD ? a.tiles_p * a.tiles_q : a.tiles_q), which = (uint32_t)b / per, in = (uint32_t)b % per;
  const ElPart part = GRAD ? el_find_part(a.offset, a.E, a.S, a.slab, (int)which) : el_find_rows(a.offset, a.E, a.S, BP, (int)which);
  if (part.expert > a.E + 1) return;
  // A part's tiles go by strips of four along P, column by column: sixteen that follow one another, on one XCD, take from four
  // rows of tiles and four columns.  (Gradient of w in bf16, row by row in runs of four on an XCD / so, us: 38 168 rows, 38 experts,
  // 384 x 1 280 82 / 70; 50 000, 7, 512 x 768 76 / 68; 12 000, 8, 1 408 x 2 048 87 / 94.)  fp32 needs an eighth of the bytes in the
  // same time and rather has its tiles spread evenly: strips of two in runs of four (30 000, 4, 768 x 768: 274 us, 325 in sixteens).
  // Tiles of a product by rows go in runs of eight (38 168, 38 experts, 1 280 to 384 bf16: 45 us, in fours 53).
  constexpr uint32_t HIGH = !GRAD ? 1 : sizeof(T) == 2 ? 4 : 2;
  const uint32_t strip = HIGH * (uint32_t)a.tiles_q, top = in / strip * HIGH;
  const uint32_t high = !GRAD ? 1 : (uint32_t)a.tiles_p - top < HIGH ? (uint32_t)a.tiles_p - top : HIGH;
  const int q0 = (int)(in % strip / high) * BQ, p0 = GRAD ? (int)(top + in % strip % high) * BP : 0;
  const int64_t e = part.expert < a.E ? part.expert : 0;
  const int batch = (int)(part.hi - part.lo);                           // rows of the batch
  const int rows_out = GRAD ? (a.rows - p0 < BP ? a.rows - p0 : BP) : batch, cols_out = a.cols - q0 < BQ ? a.cols - q0 : BQ;
  const int inner = GRAD ? batch : part.expert < a.E ? a.inner : 0;     // (rows of no expert: zeros)
  const uint32_t ld_p = GRAD ? a.rows : a.inner, ld_q = QT ? a.cols : a.inner;
  const T *pp = static_cast<const T *>(a.p) + (GRAD ? part.lo * a.rows + p0 : part.lo * a.inner);
  const T *pq = static_cast<const T *>(a.q) +
                (GRAD ? part.lo * a.cols + q0 : e * a.inner * a.cols + (KN ? (int64_t)q0 : (int64_t)q0 * a.inner));
  op_p fp;
  op_q fq;
  // bytes of a word that lie in front of the operands' first elements; every piece begins as many bytes into one
  const uint32_t skip_p = DIRECT ? 0u : reinterpret_cast<uintptr_t>(pp) & 3, skip_q = DIRECT ? 0u : reinterpret_cast<uintptr_t>(pq) & 3;
  fp.init(t, ld_p, rows_out, skip_p);
  fq.init(t, ld_q, cols_out, skip_q);
  // the operands from inner index k0 on, up to their last element (not DIRECT: in whole words)
  const auto buffer = [&](const T *p, bool outside, uint32_t ld, int wide, int k0, uint32_t skip) {
    const int left = inner - k0, n = left < BK ? left : BK;
    const uint32_t elements = outside ? (uint32_t)(n - 1) * ld + (uint32_t)wide : (uint32_t)(wide - 1) * ld + (uint32_t)left;
    const uint32_t bytes = left < 1 ? 0u : elements * SIZE;
    return hc_make_buffer(reinterpret_cast<const char *>(outside ? p + (int64_t)k0 * ld : p + k0) - skip,
                          DIRECT ? bytes : (bytes + skip + 3) & ~3u);
  };
  const auto fetch = [&](int s, int k0) {
    fp.fetch(buffer(pp, PT, ld_p, rows_out, k0, skip_p), lds + s * STAGE, t, wave, inner - k0);
    fq.fetch(buffer(pq, QT, ld_q, cols_out, k0, skip_q), lds + s * STAGE + BYTES_P, t, wave, inner - k0);
  };
  el_acc acc[TP][TQ];
#pragma unroll
  for (int i = 0; i < TP; ++i)
#pragma unroll
    for (int j = 0; j < TQ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  const auto step = [&](int from, int to, int k0, bool more) {
    el_step<op_p, op_q, TP, TQ, BYTES_P, ROWB / 32, T>(lds + from * STAGE, lds + to * STAGE, fp, fq,
                                                       buffer(pp, PT, ld_p, rows_out, k0, skip_p),
                                                       buffer(pq, QT, ld_q, cols_out, k0, skip_q), more, inner - k0, t, wave, wp,
                                                       wq, acc);
  };
  const auto put = [&](int s, int k0) {
    fp.put(lds + s * STAGE, t, inner - k0);
    fq.put(lds + s * STAGE + BYTES_P, t, inner - k0);
  };
  if (inner > 0) {
    fetch(0, 0);
    put(0, 0);
  }
  int s = 0;
  for (int k0 = 0; k0 < inner; k0 += BK) {
    // what this wave has fetched for this step is in LDS, and so, behind the barrier, is what the others have
    __builtin_amdgcn_s_waitcnt(0x0070);
    __syncthreads();
    const bool more = k0 + BK < inner;
    step(s, s ^ 1, k0 + BK, more);
    s ^= 1;
    if (more) put(s, k0 + BK);
  }
  // lane l has row l % 32 of a tile of 32 x 32 and of every eight columns the four from 4 (l / 32) on
  const int l32 = lane & 31, h = lane >> 5;
  if (GRAD && part.parts > 1) {
    float *o = a.part + (int64_t)part.place * a.rows * a.cols + (int64_t)p0 * a.cols + q0;
    const bool four = a.cols % 4 == 0;
#pragma unroll
    for (int i = 0; i < TP; ++i)
#pragma unroll
      for (int j = 0; j < TQ; ++j)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const int row = wp + i * 32 + l32, col = wq + j * 32 + r * 2 + h * 4;
          if (row < rows_out && col < cols_out) {
            float *at = o + (int64_t)row * a.cols + col;
            const float v[4] = {acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]};
            if (four) {
              hc_vec<float, 4>::store(at, v);
            } else {
#pragma unroll
              for (int x = 0; x < 4; ++x)
                if (col + x < cols_out) at[x] = v[x];
            }
          }
        }
    return;
  }
  T *out = static_cast<T *>(a.out) + (GRAD ? (e * a.rows + p0) * a.cols + q0 : part.lo * a.cols + q0);
  // a wave's 32 rows at a time through its own piece of LDS, so that a row leaves in pieces of 16 bytes
  constexpr int ROW = TQ * 32 + PER;
  static_assert(WP * WQ * 32 * ROW * (int)sizeof(T) <= MEM, "the way out fits the stages");
  __syncthreads();
  T *own = reinterpret_cast<T *>(s_mem) + wave * 32 * ROW;
#pragma unroll
  for (int i = 0; i < TP; ++i) {
#pragma unroll
    for (int j = 0; j < TQ; ++j)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const float v[4] = {acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]};
        hc_vec<T, 4>::store(own + l32 * ROW + j * 32 + r * 2 + h * 4, v);
      }
    __builtin_amdgcn_wave_barrier();
    constexpr int PIECES = TQ * 32 / PER;                  // of a row
#pragma unroll
    for (int q = 0; q < 32 * PIECES / HC_WAVE; ++q) {
      const int f = q * HC_WAVE + lane, row = f / PIECES, c = f % PIECES * PER;
      const int orow = wp + i * 32 + row, ocol = wq + c;
      if (orow < rows_out && ocol < cols_out) {
        T *o = out + (int64_t)orow * a.cols + ocol;
        if (a.whole && ocol + PER <= cols_out) {
          *reinterpret_cast<el_words *>(o) = *reinterpret_cast<const el_piece *>(own + row * ROW + c);
        } else {
#pragma unroll
          for (int x = 0; x < PER; ++x)
            if (ocol + x < cols_out) o[x] = own[row * ROW + c + x];
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The gradients of experts of several parts: their partial sums added up, a quarter of the parts by each wave in their order,
// then the quarters in order.  A lane has four adjacent values (one where VEC is 1), a block 64 lanes' of one expert at a time.
template <typename T, int VEC>
__global__ __launch_bounds__(HC_BLOCK) void el_join(ElProduct a, int64_t size, int chunks) {
  __shared__ float s_part[3][VEC][HC_WAVE];
  const int lane = hc_lane(), wave = hc_wave_in_block();
  int64_t item = blockIdx.x;                    // chunk of an expert of several parts, expert by expert
  int before = 0, most = 0;
  for (int e0 = 0; e0 < a.E; e0 += HC_WAVE) {
    int64_t lo, hi;
    el_rows_of(a.offset, a.E, a.S, e0 + lane < a.E ? e0 + lane : a.E + 1, &most, &lo, &hi);
    int parts = (int)((hi - lo + a.slab - 1) / a.slab);
    parts = parts > 1 ? parts : 0;
    const int place = before + el_scan(parts) - parts;
    uint64_t several = __ballot(parts > 0);
    for (; several != 0; several &= several - 1, item -= chunks) {
      const int l = __ffsll((long long)several) - 1, n = __builtin_amdgcn_readlane(parts, l);
      const float *p = a.part + (int64_t)__builtin_amdgcn_readlane(place, l) * size;
      T *o = static_cast<T *>(a.out) + (e0 + l) * size;
      for (; item < chunks; item += gridDim.x) {
        const int64_t at = (item * HC_WAVE + lane) * VEC;
        float s[VEC];
#pragma unroll
        for (int x = 0; x < VEC; ++x) s[x] = 0.f;
        if (at < size) {
          int q = n * wave / 4;
          const int end = n * (wave + 1) / 4;
          constexpr int FLIGHT = 4;
          for (; q + FLIGHT <= end; q += FLIGHT) {
            float v[FLIGHT][VEC];
#pragma unroll
            for (int f = 0; f < FLIGHT; ++f) hc_vec<float, VEC>::load(p + (q + f) * size + at, v[f]);
#pragma unroll
            for (int f = 0; f < FLIGHT; ++f)
#pragma unroll
              for (int x = 0; x < VEC; ++x) s[x] += v[f][x];
          }
          for (; q < end; ++q) {
            float v[VEC];
            hc_vec<float, VEC>::load(p + q * size + at, v);
#pragma unroll
            for (int x = 0; x < VEC; ++x) s[x] += v[x];
          }
        }
        if (wave > 0)
#pragma unroll
          for (int x = 0; x < VEC; ++x) s_part[wave - 1][x][lane] = s[x];
        __syncthreads();
        if (wave == 0 && at < size) {
#pragma unroll
          for (int w = 0; w < 3; ++w)
#pragma unroll
            for (int x = 0; x < VEC; ++x) s[x] += s_part[w][x][lane];
          hc_vec<T, VEC>::store(o + at, s);
        }
        __syncthreads();
      }
    }
    before = __builtin_amdgcn_readlane(place + parts, HC_WAVE - 1);
  }
}

template <typename T, int BP, int BQ, int WP, int WQ, int ROWB, bool GRAD, bool KN, bool DIRECT>
static int el_launch(ElProduct a, int64_t parts, hipStream_t st) {
  a.tiles_p = GRAD ? (a.rows + BP - 1) / BP : 1;
  a.tiles_q = (a.cols + BQ - 1) / BQ;
  const int64_t blocks = parts * a.tiles_p * a.tiles_q;
  if (!hc_grid_ok(blocks)) return HC_EUNSUPPORTED;
  el_tile<T, BP, BQ, WP, WQ, ROWB, GRAD, KN, DIRECT><<<dim3((unsigned)blocks), dim3(WP * WQ * HC_WAVE), 0, st>>>(a);
  return hc_launch_status();
}

// Do rows of these widths at these addresses start on 4 bytes?
static bool el_direct(const void *p, const void *q, int64_t w0, int64_t w1, int size) {
  return ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q) | (uint64_t)(w0 * size) | (uint64_t)(w1 * size)) & 3) == 0;
}

// Tiles of 256 x 256 on eight waves, one block per compute unit, of 128 x 128 on four, two blocks per unit, or of 64 x 64 on
// four; pieces of 128 bytes of inner index, or of 64, which leaves room for four small blocks on a unit.  (256 x 128 on four waves,
// two blocks per unit: 65 536 x 1 280 x 1 280 bf16 256 us, 222 by the large ones.)
#define EL_LARGE 256, 256, 2, 4, 128
#define EL_SMALL 128, 128, 2, 2, 128
#define EL_SHORT 128, 128, 2, 2, 64
#define EL_TINY 64, 64, 2, 2, 128
#define EL_TINY_GRAD 64, 64, 2, 2, 64

// Longest inner size that small tiles take in pieces of 64 bytes.  us, in 128 / in 64: 100 000 rows, 5 experts, 256 x 256 31 / 26;
// 20 000, 32, 512 x 512 21.0 / 20.8; 12 000, 8, 1 408 x 2 048 86 / 104.
constexpr int EL_SHORT_INNER = 512;
// 128-wide tiles of half precision up to which tiles of 64 x 64 are taken: no unit would have two (us, small / tiny: 1 000 rows, 8
// experts, 768 x 768: 10.4 / 7.7; 3 000, 16, 512 x 512: 10 / 7; 10 000, 1, 256 x 602 (158): 11.4 / 10.5; 602 x 256 (395): 10.8 / 11.5)
constexpr int64_t EL_TINY_ROWS = 256;
// Rows of an expert, on average, up to which its gradient goes in pieces of 64 bytes (half precision; us, in 128 / in 64: 16 384 rows,
// 64 experts, 768 x 1 024 75 / 58; 20 000, 32, 512 x 512 39 / 37; 8 192, 8, 1 024 x 1 024 41 / 41; 12 000, 8, 1 408 x 2 048 84 / 108).
constexpr int64_t EL_SHORT_GROUP = 640;
// Rows of the batch that a unit would take through a large tile, times the units, from which a gradient goes by large ones (us, small /
// large: 65 536 rows, 1 280 x 1 280 (25 tiles) 262 / 221; 32 771, 16 experts, 2 048 x 1 024 (32) 150 / 160).
constexpr int64_t EL_LARGE_GRAD = 256 * 5120;
// The same of a small tile in fp32, below which its gradient goes by tiny ones (us, small / tiny: 500 rows, 4 experts, 256 x 256:
// 18 / 13; 20 000, 7, 300 x 172: 47 / 36; 40 000, 1, 256 x 602: 123 / 123; 30 000, 4, 768 x 768: 274 / 289)
constexpr int64_t EL_SMALL_GRAD_F32 = 256 * 2048;

// Is the product of S rows in E groups by `cols` columns done sooner in large tiles?  Rounds over the 256 compute units, the
// groups' last tiles half empty; a small tile, two at a time on a unit, takes EL_SMALL_COST of a large one's time and does a
// quarter of its work.  (us, large / small: 65 536 rows, 1 280 x 1 280 225 / 265; 8 192, 8 192 x 1 024 134 / 145, its gradient of x
// 179 / 121; 38 168, 38 experts, 384 x 1 280 67 / 45.)
constexpr float EL_SMALL_COST = 0.575f;
static int64_t el_tiles_of_rows(int64_t S, int64_t E, int64_t cols, int64_t tile) {
  return ((S + tile - 1) / tile + E / 2) * ((cols + tile - 1) / tile);
}
static bool el_large_rows(int64_t S, int64_t E, int64_t cols) {
  const int64_t large = el_tiles_of_rows(S, E, cols, 256), small = el_tiles_of_rows(S, E, cols, 128);
  return (float)((large + 255) / 256) <= EL_SMALL_COST * (float)((small + 511) / 512);
}

// The same for fp32, tiles of 128 x 128 and of 64 x 64.  Matrix instructions of fp32 fill a unit with one tile of either kind, so
// that what counts is the rounds alone; a tiny tile takes EL_TINY_COST of a small one's time.  (us for the result, small / tiny:
// 500 rows, 4 experts, 256 x 256: 22 / 9; 9 000, 3, 1 024 x 512: 133 / 91; 20 000, 1, 602 x 256: 86 / 60; 60 007, 5, 256 x 256:
// 82 / 88; 30 000, 4, 768 x 768: 290 / 304.)
constexpr float EL_TINY_COST = 0.28f;
static bool el_small_rows_f32(int64_t S, int64_t E, int64_t cols) {
  const int64_t small = el_tiles_of_rows(S, E, cols, 128), tiny = el_tiles_of_rows(S, E, cols, 64);
  return (float)((small + 255) / 256) <= EL_TINY_COST * (float)((tiny + 255) / 256);
}

template <typename T, bool KN>
static int el_rows_of_type(const ElProduct &a, hipStream_t st) {
  const int64_t parts = a.S / 128 + a.E + 2;
  bool tiny;
  if constexpr (sizeof(T) == 2) {
    if (!el_direct(a.p, a.q, a.inner, KN ? a.cols : a.inner, 2)) return el_launch<T, EL_SHORT, false, KN, false>(a, parts, st);
    if (el_large_rows(a.S, a.E, a.cols)) return el_launch<T, EL_LARGE, false, KN, true>(a, a.S / 256 + a.E + 2, st);
    tiny = el_tiles_of_rows(a.S, a.E, a.cols, 128) <= EL_TINY_ROWS;
    if (!tiny && a.inner > EL_SHORT_INNER) return el_launch<T, EL_SMALL, false, KN, true>(a, parts, st);
  } else {
    tiny = !el_small_rows_f32(a.S, a.E, a.cols);
  }
  if (tiny) return el_launch<T, EL_TINY, false, KN, true>(a, a.S / 64 + a.E + 2, st);
  return el_launch<T, EL_SHORT, false, KN, true>(a, parts, st);
}

constexpr int EL_JOIN_BLOCKS = 2048;

struct ElGradShape {
  bool large;
  int64_t slab, several;        // rows of a part; parts of experts with several of them, at most
};

// Parts: as few as give every compute unit a large tile or two small ones, had one expert all rows (half as long, us: 50 000 rows, 7
// experts, 512 x 768 bf16 68 / 80; 30 000, 4, 768 x 768 fp32 275 / 293; 60 007, 5, 256 x 256 fp32 84 / 96).  A part has 512 rows at
// least, 128 in fp32, whose products of as many rows take eight times as long (4 000 rows, 8 experts, 256 x 256: 128 / 512 22 / 43 us;
// bf16, 3 000, 16, 512 x 512: 24 / 18).
static ElGradShape el_grad_shape(int64_t S, int64_t N, int64_t K, int size, bool wide) {
  ElGradShape g;
  const int64_t large = (N + 255) / 256 * ((K + 255) / 256), small = (N + 127) / 128 * ((K + 127) / 128);
  g.large = wide && size == 2 && S * large >= EL_LARGE_GRAD;
  const int64_t parts = g.large ? 256 / large : 512 / small;
  g.slab = (S / (parts < 1 ? 1 : parts) + 64) / 64 * 64;
  const int64_t least = size == 2 ? 512 : 128;
  if (g.slab < least) g.slab = least;
  // an expert of p > 1 parts has more than (p - 1) slab >= p / 2 slab rows
  g.several = S <= g.slab ? 0 : 2 * (S / g.slab);
  return g;
}

template <typename T>
static int el_grad_of_type(ElProduct a, void *workspace, size_t workspace_bytes, hipStream_t st) {
  const bool direct = el_direct(a.p, a.q, a.rows, a.cols, (int)sizeof(T));
  const ElGradShape g = el_grad_shape(a.S, a.rows, a.cols, (int)sizeof(T), direct);
  const int64_t size = (int64_t)a.rows * a.cols;
  if ((size_t)(g.several * size) * sizeof(float) > workspace_bytes ||
      (g.several && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)))
    return HC_EWORKSPACE;
  a.part = static_cast<float *>(workspace);
  a.slab = g.slab;
  const int64_t parts = a.S / g.slab + a.E;
  const auto run = [&]() -> int {
    if constexpr (sizeof(T) == 2) {
      if (!direct) return el_launch<T, EL_SMALL, true, false, false>(a, parts, st);
      if (g.large) return el_launch<T, EL_LARGE, true, false, true>(a, parts, st);
    }
    const int64_t small = (int64_t)((a.rows + 127) / 128) * ((a.cols + 127) / 128);
    if constexpr (sizeof(T) == 4) {
      if (a.S * small < EL_SMALL_GRAD_F32) return el_launch<T, EL_TINY_GRAD, true, false, true>(a, parts, st);
    } else {
      if (a.S <= EL_SHORT_GROUP * a.E) return el_launch<T, EL_SHORT, true, false, true>(a, parts, st);
    }
    return el_launch<T, EL_SMALL, true, false, true>(a, parts, st);
  };
  const int rc = run();
  if (rc != HC_OK || g.several == 0) return rc;
  const bool four = size % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % (4 * sizeof(T)) == 0;
  const int64_t chunks = (size + HC_WAVE * (four ? 4 : 1) - 1) / (HC_WAVE * (four ? 4 : 1));
  const int64_t most = chunks * (a.E < g.several / 2 ? a.E : g.several / 2);
  const dim3 blocks((unsigned)(most < EL_JOIN_BLOCKS ? most : EL_JOIN_BLOCKS));
  if (four) el_join<T, 4><<<blocks, dim3(HC_BLOCK), 0, st>>>(a, size, (int)chunks);
  else el_join<T, 1><<<blocks, dim3(HC_BLOCK), 0, st>>>(a, size, (int)chunks);
  return hc_launch_status();
}

}  // namespace

#define EL_FOR_TYPE(T, name)                                                                                       \
  int el_rows_##name(bool w_is_kn, const ElProduct &a, hipStream_t st) {                                           \
    return w_is_kn ? el_rows_of_type<T, true>(a, st) : el_rows_of_type<T, false>(a, st);                           \
  }                                                                                                                \
  int el_grad_##name(const ElProduct &a, void *workspace, size_t workspace_bytes, hipStream_t st) {                \
    return el_grad_of_type<T>(a, workspace, workspace_bytes, st);                                                  \
  }                                                                                                                \
  size_t el_grad_bytes_##name(int64_t S, int64_t E, int64_t N, int64_t K) {                                        \
    const int64_t wide = el_grad_shape(S, N, K, (int)sizeof(T), true).several;                                  \
    const int64_t other = el_grad_shape(S, N, K, (int)sizeof(T), false).several;                                \
    return (size_t)(wide > other ? wide : other) * (size_t)N * (size_t)K * sizeof(float);                          \
  }
