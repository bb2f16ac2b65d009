// Rows of any width and alignment by eight adjacent elements a lane, and groups of columns as 8-bit codes with an fp32 scale.
#pragma once

#include "hc_common.h"

#ifdef __HIPCC__

constexpr float PK_SMALLEST = 0x1p-120f;
constexpr float PK_LARGEST_SCALE = 0x1.0204060000000p+121f;      // 127 times the next one leaves fp32
constexpr int PK_EACH = 8;

// 16 bytes at the alignment of one element
typedef uint32_t pk_words_2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t pk_words_4 __attribute__((ext_vector_type(4), aligned(4)));
// N elements of S bytes at the alignment of one, as words
template <int S, int N>
struct pk_few {
  struct __attribute__((packed, aligned(S < 4 ? S : 4))) words {
    uint32_t w[S * N >= 4 ? S * N / 4 : 1];
  };
  struct __attribute__((packed, aligned(S < 4 ? S : 4))) half {
    uint16_t h;
  };
  __device__ __forceinline__ static void load(const char *p, uint32_t *w) {
    if constexpr (S * N >= 4) {
      const words q = *reinterpret_cast<const words *>(p);
#pragma unroll
      for (int i = 0; i < S * N / 4; ++i) w[i] = q.w[i];
    } else if constexpr (S * N == 2) {
      w[0] = reinterpret_cast<const half *>(p)->h;
    } else {
      w[0] = *reinterpret_cast<const uint8_t *>(p);
    }
  }
  __device__ __forceinline__ static void store(char *p, const uint32_t *w) {
    if constexpr (S * N >= 4) {
      words q;
#pragma unroll
      for (int i = 0; i < S * N / 4; ++i) q.w[i] = w[i];
      *reinterpret_cast<words *>(p) = q;
    } else if constexpr (S * N == 2) {
      reinterpret_cast<half *>(p)->h = (uint16_t)w[0];
    } else {
      *reinterpret_cast<uint8_t *>(p) = (uint8_t)w[0];
    }
  }
};

// The first 1 to 7 of eight elements of S bytes (2 S words, the others zeros): four, two and one at a time, as the bits of
// `valid` say.
template <int S>
__device__ __forceinline__ void pk_load_tail(const char *p, int valid, uint32_t (&w)[2 * S]) {
  uint32_t four[S] = {}, two[S] = {}, one[1] = {}, a[S] = {};
  if (valid & 4) pk_few<S, 4>::load(p, four);
  if (valid & 2) pk_few<S, 2>::load(p + (valid & 4) * S, two);
  if (valid & 1) pk_few<S, 1>::load(p + (valid & 6) * S, one);
  const bool pair = (valid & 2) != 0;
  if constexpr (S == 1) {
    a[0] = two[0] | one[0] << (pair ? 16 : 0);
  } else {
    a[0] = pair ? two[0] : one[0];
    if constexpr (S == 4) a[1] = two[1];
    a[S / 2] = pair ? one[0] : 0u;
  }
#pragma unroll
  for (int i = 0; i < S; ++i) {
    w[i] = valid & 4 ? four[i] : a[i];
    w[S + i] = valid & 4 ? a[i] : 0u;
  }
}

template <int S>
__device__ __forceinline__ void pk_store_tail(char *p, int valid, const uint32_t (&w)[2 * S]) {
  uint32_t a[S];
#pragma unroll
  // (by bits: a choice between neighbours becomes a search by a computed index)
  for (int i = 0; i < S; ++i) a[i] = w[i] ^ ((w[i] ^ w[S + i]) & (valid & 4 ? ~0u : 0u));
  if (valid & 4) pk_few<S, 4>::store(p, w);
  if (valid & 2) pk_few<S, 2>::store(p + (valid & 4) * S, a);
  const uint32_t one = valid & 2 ? (S == 1 ? a[0] >> 16 : a[S / 2]) : a[0];
  if (valid & 1) pk_few<S, 1>::store(p + (valid & 6) * S, &one);
}

// Eight adjacent elements, at no more than their own alignment; those behind `valid` read as zeros and are not written.
template <typename T>
struct pk_row {
  typedef typename std::conditional<sizeof(T) == 2, pk_words_2, pk_words_4>::type words;
  static constexpr int S = (int)sizeof(T), PIECES = S * PK_EACH / 16;
  union eight {
    words q[PIECES];
    uint32_t w[2 * S];
    T e[PK_EACH];
    __device__ eight() {}
  };
  __device__ __forceinline__ static void load(const T *__restrict__ p, int valid, float (&v)[PK_EACH]) {
    eight x;
    if (valid >= PK_EACH) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) x.q[i] = reinterpret_cast<const words *>(p)[i];
    } else if (valid > 0) {
      pk_load_tail<S>(reinterpret_cast<const char *>(p), valid, x.w);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * S; ++i) x.w[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < PK_EACH; ++i) v[i] = hc_to_f32<T>(x.e[i]);
  }
  // NT: with the non-temporal hint
  template <bool NT = false>
  __device__ __forceinline__ static void store(T *__restrict__ p, int valid, const float (&v)[PK_EACH]) {
    eight x;
#pragma unroll
    for (int i = 0; i < PK_EACH; ++i) x.e[i] = hc_from_f32<T>(v[i]);
    if (valid >= PK_EACH) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        words *at = reinterpret_cast<words *>(p) + i;
        if (NT) __builtin_nontemporal_store(x.q[i], at);
        else *at = x.q[i];
      }
    } else if (valid > 0) {
      pk_store_tail<S>(reinterpret_cast<char *>(p), valid, x.w);
    }
  }
};

struct __attribute__((packed, aligned(1))) pk_codes {
  uint32_t w[2];
};

__device__ __forceinline__ void pk_load_codes(const int8_t *__restrict__ p, int valid, float scale, float (&v)[PK_EACH]) {
  uint32_t w[2];
  if (valid >= PK_EACH) {
    const pk_codes q = *reinterpret_cast<const pk_codes *>(p);
    w[0] = q.w[0];
    w[1] = q.w[1];
  } else {
    pk_load_tail<1>(reinterpret_cast<const char *>(p), valid, w);
  }
#pragma unroll
  for (int i = 0; i < PK_EACH; ++i) v[i] = (float)(int8_t)(w[i / 4] >> (8 * (i % 4))) * scale;
}

// NT: with the non-temporal hint
template <bool NT = false>
__device__ __forceinline__ void pk_store_codes(int8_t *__restrict__ p, int valid, const uint32_t (&w)[2]) {
  if (valid >= PK_EACH) {
    if constexpr (NT) {
      typedef uint32_t two __attribute__((ext_vector_type(2), aligned(1)));
      __builtin_nontemporal_store(two{w[0], w[1]}, reinterpret_cast<two *>(p));
    } else {
      *reinterpret_cast<pk_codes *>(p) = pk_codes{{w[0], w[1]}};
    }
  } else if (valid > 0) {
    pk_store_tail<1>(reinterpret_cast<char *>(p), valid, w);
  }
}

// The scale of the group that L lanes hold, and this lane's codes.  The largest magnitude is found on the bits, where a NaN
// is above infinity and infinity above every number.
template <int L>
__device__ __forceinline__ float pk_encode(const float (&v)[PK_EACH], uint32_t (&w)[2]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < PK_EACH; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  m = hc_join<L>(m, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
  const float most = __uint_as_float(m);
  const bool zero = most < PK_SMALLEST, bad = m >= 0x7f800000u;
  const float inverse = zero || bad ? 0.f : 1.0f / most * 127.0f;
  // 1.5 2^23 more has the rounded number in its lowest byte
  uint32_t c[PK_EACH];
#pragma unroll
  for (int i = 0; i < PK_EACH; ++i) c[i] = __float_as_uint(v[i] * inverse + 0x1.8p23f);
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[4 * i + 3], c[4 * i + 2], 0x0c0c0400u),
                                 __builtin_amdgcn_perm(c[4 * i + 1], c[4 * i], 0x0c0c0400u), 0x05040100u);
  if (bad) w[0] = w[1] = 0;
  const float scale = most * (1.0f / 127.0f);
  return zero ? 0.f : !bad && scale > PK_LARGEST_SCALE ? PK_LARGEST_SCALE : scale;
}

template <int L>
__device__ __forceinline__ float pk_encode(const float (&v)[PK_EACH], int8_t *__restrict__ p, int valid) {
  uint32_t w[2];
  const float scale = pk_encode<L>(v, w);
  pk_store_codes(p, valid, w);
  return scale;
}

#endif  // __HIPCC__
