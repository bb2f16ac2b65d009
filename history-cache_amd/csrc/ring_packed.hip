// Lookup in a ring table of embeddings held in 8 bits (packed_rows.h): slots of ids, and the hits' rows in fp32, code * scale.
//
// A block takes a few rows: its first lanes look a row up each (three reads that wait for one another), then all of its lanes lie
// one after the other over the rows' columns.
#include "packed_rows.h"

namespace {

constexpr int RP_MOST_ROWS = 64;       // rows a block

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
// any alignment.
template <int V>
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
    const int64_t slot = s_slot[r];
    const uint32_t col = c * V;
    float *out = a.rows_out + (row0 + r) * a.F + col;
    if constexpr (V == 4) {
      uint32_t w = 0;
      float s = 0.f;
      if (slot >= 0) {
        w = *reinterpret_cast<const uint32_t *>(a.codes + slot * a.F + col);
        s = a.scale[slot * a.groups + col / a.group];
      }
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = (float)(int8_t)(w >> (8 * i)) * s;
      if (slot < 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.f;
      }
      hc_vec<float, V>::store(out, v);
    } else {
      const int valid = a.F - col >= (uint32_t)PK_EACH ? PK_EACH : (int)(a.F - col);
      float v[PK_EACH];
#pragma unroll
      for (int i = 0; i < PK_EACH; ++i) v[i] = 0.f;
      if (slot >= 0) pk_load_codes(a.codes + slot * a.F + col, valid, a.scale[slot * a.groups + col / a.group], v);
      pk_row<float>::store(out, valid, v);
    }
    r += down;
    c += across;
    if (c >= pieces) c -= pieces, ++r;
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
  const int64_t blocks = (n + a.rows - 1) / a.rows;
  if (!hc_grid_ok(blocks)) return HC_EUNSUPPORTED;
  const bool whole = F % 4 == 0 && reinterpret_cast<uintptr_t>(codes) % 4 == 0 && reinterpret_cast<uintptr_t>(rows_out) % 16 == 0;
  const auto kernel = whole ? rp_lookup<4> : rp_lookup<8>;
  kernel<<<dim3((unsigned)blocks), dim3(HC_BLOCK), 0, static_cast<hipStream_t>(stream)>>>(a);
  return hc_launch_status();
}
