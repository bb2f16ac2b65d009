// Lookup in a ring table of embeddings held in 8 bits (packed_rows.h): slots of ids, and the hits' rows in fp32, code * scale.
//
// A block takes 16 rows, in large calls 64: its first lanes look a row up each (three reads that wait for one another), then all of its
// lanes lie one after the other over the rows' columns.
// Bound by memory where there are many: 1 000 003 ids, 400 000 of them hits of 256 columns, 243 us for 1.15 GB (4.7 TB/s; an id's map
// entry, age, scales and codes lie in lines of their own, 0.25 GB more than is asked for; from a table in fp16 501 us).  With ordinary
// stores 291; one, two or four pieces at once 379, 268 and 266 (maps in the last-level cache); eight, or the next pieces read before the
// last are written, as four.  16 rows a block 264, behind an admission of as many rows, which leaves the maps in memory: the three
// reads of a block's start then take longer than 16 rows do (with the maps in the cache, from one lookup to the next, it is
// the other way round, 266 against 281).  1 500 ids of 128 columns 2.8 with 16 rows, 3.8 with 64.
// 150 001 ids, half of them hits of 172 columns: 27 us (118 MB) either way.  Few: 8 661 of 256 columns 5.4, 1 500 of 128 3.9 us, a launch
// and four reads one after the other.
#include "packed_rows.h"

namespace {

constexpr int RP_MOST_ROWS = 64;       // rows a block
constexpr int RP_AT_ONCE = 4;          // pieces that a lane reads before it writes the first
constexpr int64_t RP_CACHE = 256 << 20;          // bytes of the last-level cache

struct RpArgs {
  const int64_t *full2slot, *ids, *checkin, *now_dev, *n_valid_dev;
  int64_t n_full, now, age_limit, capacity, n;
  const int8_t *codes;
  const float *scale;
  int64_t *slot_out;
  float *rows_out;
  uint32_t F, groups, group, rows;
};

__device__ __forceinline__ int64_t rp_find(const RpArgs &a, int64_t i) {
  const int64_t now = a.now_dev != nullptr ? *a.now_dev : a.now;
  const bool padding = a.n_valid_dev != nullptr && i >= *a.n_valid_dev;
  const int64_t id = padding ? -1 : a.ids[i];
  int64_t slot = id >= 0 && id < a.n_full ? a.full2slot[id] : -1;
  if (slot < 0 || slot >= a.capacity) return -1;
  if (a.checkin != nullptr && now - a.checkin[slot] >= a.age_limit) return -1;
  return slot;
}

// V: adjacent columns a lane: 4 where rows are whole multiples of four columns and lie at multiples of 16 bytes, otherwise 8 at
// any alignment.  NT: for rows that the last-level cache cannot hold until they are read.
template <int V, bool NT>
__global__ __launch_bounds__(HC_BLOCK) void rp_lookup(RpArgs a) {
  __shared__ int64_t s_slot[RP_MOST_ROWS];
  const int64_t row0 = (int64_t)blockIdx.x * a.rows;
  const uint32_t rows = a.n - row0 < (int64_t)a.rows ? (uint32_t)(a.n - row0) : a.rows;
  if (threadIdx.x < rows) {
    const int64_t slot = rp_find(a, row0 + threadIdx.x);
    s_slot[threadIdx.x] = slot;
    a.slot_out[row0 + threadIdx.x] = slot;
  }
  if (a.rows_out == nullptr) return;
  __syncthreads();
  const uint32_t pieces = (a.F + V - 1) / V, down = HC_BLOCK / pieces, across = HC_BLOCK % pieces;
  uint32_t r = threadIdx.x / pieces, c = threadIdx.x % pieces;
  while (r < rows) {
    uint32_t w[RP_AT_ONCE][2], row_of[RP_AT_ONCE], col_of[RP_AT_ONCE];
    float s[RP_AT_ONCE];
#pragma unroll
    for (int u = 0; u < RP_AT_ONCE; ++u) {
      row_of[u] = r;
      col_of[u] = c * V;
      w[u][0] = w[u][1] = 0;
      s[u] = 0.f;
      const int64_t slot = r < rows ? s_slot[r] : -1;
      if (slot >= 0) {
        const int8_t *from = a.codes + slot * a.F + col_of[u];
        s[u] = a.scale[slot * a.groups + col_of[u] / a.group];
        if constexpr (V == 4) {
          w[u][0] = *reinterpret_cast<const uint32_t *>(from);
        } else {
          const int valid = a.F - col_of[u] >= (uint32_t)PK_EACH ? PK_EACH : (int)(a.F - col_of[u]);
          if (valid >= PK_EACH) {
            const pk_codes q = *reinterpret_cast<const pk_codes *>(from);
            w[u][0] = q.w[0];
            w[u][1] = q.w[1];
          } else {
            pk_load_tail<1>(reinterpret_cast<const char *>(from), valid, w[u]);
          }
        }
      }
      r += down;
      c += across;
      if (c >= pieces) c -= pieces, ++r;
    }
#pragma unroll
    for (int u = 0; u < RP_AT_ONCE; ++u) {
      if (row_of[u] >= rows) break;
      float *out = a.rows_out + (row0 + row_of[u]) * a.F + col_of[u];
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = (float)(int8_t)(w[u][i / 4] >> (8 * (i % 4))) * s[u];
      if constexpr (V == 4) {
        if constexpr (NT) hc_vec<float, 4>::store_nt(out, v);
        else hc_vec<float, 4>::store(out, v);
      } else {
        const int valid = a.F - col_of[u] >= (uint32_t)PK_EACH ? PK_EACH : (int)(a.F - col_of[u]);
        pk_row<float>::template store<NT>(out, valid, v);
      }
    }
  }
}

}  // namespace

extern "C" int hc_ring_lookup_packed(const int64_t *full2slot, int64_t n_full, const int64_t *ids, const int64_t *checkin,
                                     int64_t now, const int64_t *now_dev, const int64_t *n_valid_dev, int64_t age_limit,
                                     const int8_t *codes, const float *scale, int64_t group, int64_t capacity, int64_t F,
                                     int64_t *slot_out, float *rows_out, int64_t n, void *stream) {
  HC_REQUIRE(n >= 0 && n_full >= 0 && capacity >= 0 && F > 0);
  if ((group != 32 && group != 64 && group != 128) || F >= (1 << 30)) return HC_EUNSUPPORTED;
  if (n == 0) return HC_OK;
  HC_REQUIRE(full2slot && ids && slot_out);
  HC_REQUIRE(rows_out == nullptr || (codes && scale));
  RpArgs a{full2slot, ids, checkin, now_dev, n_valid_dev, n_full, now, age_limit, capacity, n, codes, scale, slot_out, rows_out,
           (uint32_t)F, (uint32_t)((F + group - 1) / group), (uint32_t)group, 16};
  a.rows = n >= 2048 * RP_MOST_ROWS ? RP_MOST_ROWS : 16;
  const int64_t blocks = (n + a.rows - 1) / a.rows;
  if (!hc_grid_ok(blocks)) return HC_EUNSUPPORTED;
  const bool whole = F % 4 == 0 && reinterpret_cast<uintptr_t>(codes) % 4 == 0 && reinterpret_cast<uintptr_t>(rows_out) % 16 == 0;
  const bool large = n * F * (int64_t)sizeof(float) > RP_CACHE;
  const auto kernel = whole ? (large ? rp_lookup<4, true> : rp_lookup<4, false>) : large ? rp_lookup<8, true> : rp_lookup<8, false>;
  kernel<<<dim3((unsigned)blocks), dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(a);
  return hc_launch_status();
}
