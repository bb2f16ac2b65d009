// Rows times their expert's matrix in fp16 and bf16, on the matrix cores, sums in fp32.
#include "expert_find.h"

namespace {

typedef float eh_acc __attribute__((ext_vector_type(16)));
typedef short eh_frag __attribute__((ext_vector_type(8)));
typedef short eh_quad __attribute__((ext_vector_type(4)));
typedef uint32_t eh_piece __attribute__((ext_vector_type(4)));

constexpr int EH_BK = 64;                       // inner columns of a piece
constexpr uint32_t EH_NOWHERE = 0xfffffff0u;    // behind every buffer: reads as zero
#define EH_LDS __attribute__((address_space(3)))

template <typename T>
__device__ __forceinline__ eh_acc eh_mfma(eh_frag a, eh_frag b, eh_acc c) {
  if constexpr (std::is_same<T, __half>::value) {
    typedef _Float16 f16 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16, a), __builtin_bit_cast(f16, b), c, 0, 0, 0);
  } else {
    typedef __bf16 b16 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16, a), __builtin_bit_cast(b16, b), c, 0, 0, 0);
  }
}

// A piece of an operand in LDS: W rows (or columns) of the result by EH_BK inner ones, in chunks of 8 elements.
//   TR = false: inner index along memory, [W][64]; chunk c of row r lies at c ^ (r & 7), so that the eight rows that are read at
//               a time lie in different banks
//   TR = true:  inner index outside, [64][W]; read by ds_read_b64_tr_b16, 4 rows x 16 columns by 16 lanes; columns 16 c ..
//               of row r lie at c ^ (r & 7)
// PIECE = 8: chunks go straight into LDS, which takes rows and columns that start on 16 bytes; else they are loaded in pieces of
// PIECE elements, which may end inside a chunk, and pass through registers.
template <int W, bool TR, int THREADS, int PIECE>
struct eh_operand {
  static constexpr int CHUNKS = W * EH_BK / 8, EACH = CHUNKS / THREADS;
  static_assert(CHUNKS % THREADS == 0, "whole chunks per thread");
  uint32_t at[EACH];        // byte offset of this thread's chunks in the operand's first piece
  int first[EACH];          // first inner index (TR = false) or column of each
  eh_piece held[PIECE == 8 ? 1 : EACH];
  int width;

  // stride: of the operand's rows in elements; wide: rows (TR = false) or columns (TR = true) that exist from the tile's first on
  __device__ __forceinline__ void init(int t, uint32_t stride, int wide) {
    width = wide;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int q = i * THREADS + t;
      if constexpr (!TR) {
        const int r = q / 8, c = (q % 8) ^ (r & 7);
        first[i] = c * 8;
        at[i] = r < wide ? ((uint32_t)r * stride + (uint32_t)c * 8u) * 2u : EH_NOWHERE;
      } else {
        const int r = q / (W / 8), p = q % (W / 8), c = ((p / 2) ^ (r & 7)) * 2 + p % 2;
        first[i] = c * 8;
        at[i] = c * 8 < wide ? ((uint32_t)r * stride + (uint32_t)c * 8u) * 2u : EH_NOWHERE;
      }
    }
  }
  // left: inner indices from the piece's first on
  __device__ __forceinline__ void fetch(hc_buffer b, EH_LDS char *lds, int wave, int left) {
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      if constexpr (PIECE == 8) {
        const uint32_t o = TR || first[i] < left ? at[i] : EH_NOWHERE;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(b, (EH_LDS void *)(lds + (i * THREADS + wave * HC_WAVE) * 16), 16, o, 0, 0, 0);
      } else {
        const int end = TR ? width : left;
#pragma unroll
        for (int p = 0; p < 8; p += PIECE) {
          const uint32_t o = first[i] + p < end && at[i] != EH_NOWHERE ? at[i] + 2u * p : EH_NOWHERE;
          if constexpr (PIECE == 4) {
            const auto v = __builtin_amdgcn_raw_buffer_load_b64(b, o, 0, 0);
            held[i][p / 2] = v[0];
            held[i][p / 2 + 1] = v[1];
          } else if constexpr (PIECE == 2) {
            held[i][p / 2] = __builtin_amdgcn_raw_buffer_load_b32(b, o, 0, 0);
          } else {
            const uint32_t v = __builtin_amdgcn_raw_buffer_load_b16(b, o, 0, 0);
            held[i][p / 2] = p % 2 == 0 ? v : held[i][p / 2] | v << 16;
          }
        }
      }
    }
  }
  __device__ __forceinline__ void put(EH_LDS char *lds, int t) const {
    if constexpr (PIECE != 8)
#pragma unroll
      for (int i = 0; i < EACH; ++i) *(EH_LDS eh_piece *)(lds + (i * THREADS + t) * 16) = held[i];
  }
};

// The fragment of 32 rows (columns) from `first` on and inner indices 16 k ..: lane l has row first + l % 32, inner 8 (l / 32) ...
template <int W, bool TR>
__device__ __forceinline__ eh_frag eh_read(const EH_LDS char *lds, int first, int k) {
  const int lane = hc_lane();
  if constexpr (!TR) {
    const int r = first + (lane & 31), c = k * 2 + (lane >> 5);
    return *(const EH_LDS eh_frag *)(lds + r * 128 + ((c ^ (lane & 7)) * 16));
  } else {
    const int i = lane & 15, g = lane >> 4;
    const int r = k * 16 + (g >> 1) * 8 + (i >> 2), c = first / 16 + (g & 1);
    const EH_LDS char *p = lds + r * (W * 2) + (i & 3) * 8;
    const eh_quad a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((EH_LDS eh_quad *)(p + ((c ^ (i >> 2)) * 32)));
    const eh_quad b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((EH_LDS eh_quad *)(p + 4 * (W * 2) + ((c ^ ((i >> 2) + 4)) * 32)));
    return eh_frag{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
}

// GRAD: P and Q are both read with the inner index (rows of the batch) outside; else P's rows are the batch's, and KN says how Q
// lies.
template <typename T, int BP, int BQ, int WP, int WQ, bool GRAD, bool KN, int PIECE>
__global__ __launch_bounds__(WP *WQ *HC_WAVE, 2) void eh_tile(ElProduct a) {
  constexpr int THREADS = WP * WQ * HC_WAVE, TP = BP / WP / 32, TQ = BQ / WQ / 32;
  constexpr bool PT = GRAD, QT = GRAD || KN;
  typedef eh_operand<BP, PT, THREADS, PIECE> op_p;
  typedef eh_operand<BQ, QT, THREADS, PIECE> op_q;
  constexpr int BYTES_P = BP * EH_BK * 2, BYTES_Q = BQ * EH_BK * 2;
  constexpr int STAGE = BYTES_P + BYTES_Q;
  __shared__ __attribute__((aligned(16))) char s_mem[2 * STAGE];
  const int64_t b = hc_xcd_block<32>(blockIdx.x, gridDim.x);
  const int t = (int)threadIdx.x, lane = hc_lane(), wave = hc_wave_in_block();
  const int wp = wave % WP * (BP / WP), wq = wave / WP * (BQ / WQ);
  const int per = GRAD ? a.tiles_p * a.tiles_q : a.tiles_q, in = (int)(b % per);
  const ElPart part = el_find<!GRAD>(a.offset, a.E, a.S, GRAD ? a.slab : BP, (int)(b / per));
  if (part.expert > a.E) return;
  const int q0 = in % a.tiles_q * BQ, p0 = GRAD ? in / a.tiles_q * BP : 0;
  const int64_t e = part.expert < a.E ? part.expert : 0;
  const int batch = (int)(part.hi - part.lo);                           // rows of the batch
  const int rows_out = GRAD ? (a.rows - p0 < BP ? a.rows - p0 : BP) : batch, cols_out = a.cols - q0 < BQ ? a.cols - q0 : BQ;
  const int inner = GRAD ? batch : part.expert < a.E ? a.inner : 0;
  const uint32_t ld_p = GRAD ? a.rows : a.inner, ld_q = QT ? a.cols : a.inner;
  const uint16_t *pp = static_cast<const uint16_t *>(a.p) + (GRAD ? part.lo * a.rows + p0 : part.lo * a.inner);
  const uint16_t *pq = static_cast<const uint16_t *>(a.q) +
                       (GRAD ? part.lo * a.cols + q0 : e * a.inner * a.cols + (KN ? (int64_t)q0 : (int64_t)q0 * a.inner));
  op_p fp;
  op_q fq;
  fp.init(t, ld_p, rows_out);
  fq.init(t, ld_q, cols_out);
  EH_LDS char *lds = (EH_LDS char *)s_mem;
  const auto fetch = [&](int s, int k0) {
    const int left = inner - k0, n = left < EH_BK ? left : EH_BK;
    // a buffer ends with the last row that exists
    const hc_buffer bp = hc_make_buffer(PT ? pp + (int64_t)k0 * ld_p : pp + k0,
                                        PT ? ((uint32_t)(n - 1) * ld_p + (uint32_t)rows_out) * 2u : 0xffffff00u);
    const hc_buffer bq = hc_make_buffer(QT ? pq + (int64_t)k0 * ld_q : pq + k0,
                                        QT ? ((uint32_t)(n - 1) * ld_q + (uint32_t)cols_out) * 2u : 0xffffff00u);
    fp.fetch(bp, lds + s * STAGE, wave, left);
    fq.fetch(bq, lds + s * STAGE + BYTES_P, wave, left);
  };
  eh_acc acc[TP][TQ];
#pragma unroll
  for (int i = 0; i < TP; ++i)
#pragma unroll
    for (int j = 0; j < TQ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  const auto compute = [&](int s) {
#pragma unroll
    for (int k = 0; k < EH_BK / 16; ++k) {
      eh_frag u[TP], v[TQ];
#pragma unroll
      for (int i = 0; i < TP; ++i) u[i] = eh_read<BP, PT>(lds + s * STAGE, wp + i * 32, k);
#pragma unroll
      for (int j = 0; j < TQ; ++j) v[j] = eh_read<BQ, QT>(lds + s * STAGE + BYTES_P, wq + j * 32, k);
#pragma unroll
      for (int i = 0; i < TP; ++i)
#pragma unroll
        for (int j = 0; j < TQ; ++j) acc[i][j] = eh_mfma<T>(v[j], u[i], acc[i][j]);
    }
  };
  const auto put = [&](int s) {
    fp.put(lds + s * STAGE, t);
    fq.put(lds + s * STAGE + BYTES_P, t);
  };
  if (inner > 0) {
    fetch(0, 0);
    put(0);
  }
  int s = 0;
  for (int k0 = 0; k0 < inner; k0 += EH_BK) {
    __builtin_amdgcn_s_waitcnt(0x0f70);                                // vmcnt 0: what this wave has fetched is in LDS
    __syncthreads();
    const bool more = k0 + EH_BK < inner;
    if (more) fetch(s ^ 1, k0 + EH_BK);
    __builtin_amdgcn_sched_barrier(0);
    compute(s);
    s ^= 1;
    if (more) put(s);
  }
  // lane l has row l % 32 of a tile of 32 x 32 and of every eight columns the four from 4 (l / 32) on
  const int l32 = lane & 31, h = lane >> 5;
  if (GRAD && part.parts > 1) {
    float *o = a.part + (int64_t)part.place * a.rows * a.cols + (int64_t)p0 * a.cols + q0;
#pragma unroll
    for (int i = 0; i < TP; ++i)
#pragma unroll
      for (int j = 0; j < TQ; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = wp + i * 32 + l32, col = wq + j * 32 + r / 4 * 8 + h * 4 + r % 4;
          if (row < rows_out && col < cols_out) o[(int64_t)row * a.cols + col] = acc[i][j][r];
        }
    return;
  }
  T *out = static_cast<T *>(a.out) + (GRAD ? (e * a.rows + p0) * a.cols + q0 : part.lo * a.cols + q0);
  // a wave's 32 rows at a time through its own piece of LDS, so that a row leaves in pieces of 16 bytes
  constexpr int ROW = TQ * 32 + 8;
  static_assert(WP * WQ * 32 * ROW * 2 <= BYTES_P + BYTES_Q, "the way out fits a stage");
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
    constexpr int PER = TQ * 4;                       // pieces of a row
#pragma unroll
    for (int s = 0; s < 32 * PER / HC_WAVE; ++s) {
      const int f = s * HC_WAVE + lane, row = f / PER, c = f % PER * 8;
      const int orow = wp + i * 32 + row, ocol = wq + c;
      const eh_piece v = *reinterpret_cast<const eh_piece *>(own + row * ROW + c);
      if (orow < rows_out && ocol < cols_out) {
        T *o = out + (int64_t)orow * a.cols + ocol;
        if (a.whole) {
          *reinterpret_cast<eh_piece *>(o) = v;
        } else {
#pragma unroll
          for (int x = 0; x < 8; ++x)
            if (ocol + x < cols_out) o[x] = own[row * ROW + c + x];
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The gradients of experts of several parts: their partial sums added in the order of the parts.
template <typename T>
__global__ __launch_bounds__(HC_BLOCK) void eh_join(ElProduct a, int64_t size, int64_t pieces) {
  const int lane = hc_lane();
  int before = 0;
  for (int e0 = 0; e0 < a.E; e0 += HC_WAVE) {
    int64_t lo, hi;
    el_rows_of(a.offset, a.E, a.S, e0 + lane < a.E ? e0 + lane : a.E + 1, &lo, &hi);
    int parts = (int)((hi - lo + a.slab - 1) / a.slab);
    parts = parts > 1 ? parts : 0;
    const int first = before + el_scan(parts) - parts;
    uint64_t several = __ballot(parts > 0);
    while (several != 0) {
      const int l = __ffsll((long long)several) - 1;
      several &= several - 1;
      const int n = __builtin_amdgcn_readlane(parts, l);
      const float *p = a.part + (int64_t)__builtin_amdgcn_readlane(first, l) * size;
      T *o = static_cast<T *>(a.out) + (e0 + l) * size;
      for (int64_t i = (int64_t)blockIdx.x * HC_BLOCK + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * HC_BLOCK) {
        const int64_t at = i * 4;
        if (at + 4 <= size && size % 4 == 0) {
          float4 s = *reinterpret_cast<const float4 *>(p + at);
          for (int q = 1; q < n; ++q) {
            const float4 v = *reinterpret_cast<const float4 *>(p + q * size + at);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
          }
          const float v[4] = {s.x, s.y, s.z, s.w};
          if (a.whole) hc_vec<T, 4>::store(o + at, v);
          else
            for (int x = 0; x < 4; ++x) o[at + x] = hc_from_f32<T>(v[x]);
        } else {
          for (int x = 0; x < 4 && at + x < size; ++x) {
            float s = p[at + x];
            for (int q = 1; q < n; ++q) s += p[q * size + at + x];
            o[at + x] = hc_from_f32<T>(s);
          }
        }
      }
    }
    before = __builtin_amdgcn_readlane(first + parts, HC_WAVE - 1);
  }
}

template <typename T, int BP, int BQ, int WP, int WQ, bool GRAD, bool KN, int PIECE>
static int eh_launch(ElProduct a, int64_t parts, hipStream_t st) {
  a.tiles_p = GRAD ? (a.rows + BP - 1) / BP : 1;
  a.tiles_q = (a.cols + BQ - 1) / BQ;
  const int64_t blocks = parts * a.tiles_p * a.tiles_q;
  if (!hc_grid_ok(blocks)) return HC_EUNSUPPORTED;
  eh_tile<T, BP, BQ, WP, WQ, GRAD, KN, PIECE><<<dim3((unsigned)blocks), dim3(WP * WQ * HC_WAVE), 0, st>>>(a);
  return hc_launch_status();
}

// Elements in a piece that rows of these widths at these addresses allow.
static int eh_piece_of(const void *p, const void *q, int64_t w0, int64_t w1) {
  const uint64_t a = reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q) | (uint64_t)w0 * 2 | (uint64_t)w1 * 2;
  return a % 16 == 0 ? 8 : a % 8 == 0 ? 4 : a % 4 == 0 ? 2 : 1;
}

#ifndef EH_BIG
#define EH_BIG(tiles) ((tiles) >= 192)
#endif

template <typename T, bool KN>
static int eh_rows(const ElProduct &a, hipStream_t st) {
  const int piece = eh_piece_of(a.p, a.q, a.inner, KN ? a.cols : a.inner);
  const int64_t big = (a.S + 255) / 256 * ((a.cols + 255) / 256);
  if (piece == 8 && EH_BIG(big)) return eh_launch<T, 256, 256, 2, 4, false, KN, 8>(a, a.S / 256 + a.E + 1, st);
  const int64_t parts = a.S / 128 + a.E + 1;
  if (piece == 8) return eh_launch<T, 128, 128, 2, 2, false, KN, 8>(a, parts, st);
  if (piece == 4) return eh_launch<T, 128, 128, 2, 2, false, KN, 4>(a, parts, st);
  if (piece == 2) return eh_launch<T, 128, 128, 2, 2, false, KN, 2>(a, parts, st);
  return eh_launch<T, 128, 128, 2, 2, false, KN, 1>(a, parts, st);
}

struct EhGrad {
  bool big;
  int64_t slab, several;        // rows of a part; parts of experts with several of them, at most
};

static EhGrad eh_grad_shape(int64_t S, int64_t E, int64_t N, int64_t K, bool wide) {
  EhGrad g;
  const int64_t tiles = (N + 255) / 256 * ((K + 255) / 256), small = (N + 127) / 128 * ((K + 127) / 128);
  g.big = wide && EH_BIG(tiles * E);
  const int64_t want = g.big ? 256 : 1024, have = g.big ? tiles : small;
  g.slab = (S * have / want + EH_BK - 1) / EH_BK * EH_BK;
  if (g.slab < 512) g.slab = 512;
  // an expert of p > 1 parts has more than (p - 1) slab >= p / 2 slab rows
  g.several = S <= g.slab ? 0 : 2 * (S / g.slab);
  return g;
}

template <typename T>
static int eh_grad(ElProduct a, const EhGrad &g, int piece, hipStream_t st) {
  a.slab = g.slab;
  const int64_t parts = a.S / g.slab + a.E;
  int rc;
  if (g.big) rc = eh_launch<T, 256, 256, 2, 4, true, false, 8>(a, parts, st);
  else if (piece == 8) rc = eh_launch<T, 128, 128, 2, 2, true, false, 8>(a, parts, st);
  else if (piece == 4) rc = eh_launch<T, 128, 128, 2, 2, true, false, 4>(a, parts, st);
  else if (piece == 2) rc = eh_launch<T, 128, 128, 2, 2, true, false, 2>(a, parts, st);
  else rc = eh_launch<T, 128, 128, 2, 2, true, false, 1>(a, parts, st);
  if (rc != HC_OK || g.several == 0) return rc;
  const int64_t size = (int64_t)a.rows * a.cols, pieces = (size + 3) / 4;
  int64_t blocks = (pieces + HC_BLOCK - 1) / HC_BLOCK;
  blocks = blocks > 2048 ? 2048 : blocks;
  a.whole = reinterpret_cast<uintptr_t>(a.out) % 8 == 0;
  eh_join<T><<<dim3((unsigned)blocks), dim3(HC_BLOCK), 0, st>>>(a, size, pieces);
  return hc_launch_status();
}

}  // namespace

int el_half_rows(int dtype, bool w_is_kn, ElProduct a, hipStream_t st) {
  a.whole = a.cols % 8 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
  if (dtype == HC_F16) return w_is_kn ? eh_rows<__half, true>(a, st) : eh_rows<__half, false>(a, st);
  return w_is_kn ? eh_rows<__hip_bfloat16, true>(a, st) : eh_rows<__hip_bfloat16, false>(a, st);
}

// (a larger workspace than an unaligned call needs: its tiles are the smaller ones)
size_t el_half_grad_bytes(int64_t S, int64_t E, int64_t N, int64_t K) {
  const int64_t a = eh_grad_shape(S, E, N, K, true).several, b = eh_grad_shape(S, E, N, K, false).several;
  return (size_t)(a > b ? a : b) * (size_t)N * (size_t)K * sizeof(float);
}

int el_half_grad(int dtype, ElProduct a, void *workspace, size_t workspace_bytes, hipStream_t st) {
  const int piece = eh_piece_of(a.p, a.q, a.rows, a.cols);
  const EhGrad g = eh_grad_shape(a.S, a.E, a.rows, a.cols, piece == 8);
  if ((size_t)g.several * a.rows * a.cols * sizeof(float) > workspace_bytes ||
      (g.several && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)))
    return HC_EWORKSPACE;
  a.part = static_cast<float *>(workspace);
  a.whole = a.cols % 8 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
  return dtype == HC_F16 ? eh_grad<__half>(a, g, piece, st) : eh_grad<__hip_bfloat16>(a, g, piece, st);
}
