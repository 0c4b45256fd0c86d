// Pieces of eight consecutive elements of a row, at any alignment: global memory takes 16-byte accesses at every
// address, and a piece that lies on a 16-byte border costs what it always does.  Only the end of a row whose length is
// no multiple of eight goes element by element.
#pragma once
#include "common.h"

namespace cummhip {

struct F32 {};
template <> struct Elem<F32> {
  static constexpr int kBytes = 4;
};

typedef int v4i_any __attribute__((ext_vector_type(4), aligned(2)));
typedef int v4i_any1 __attribute__((ext_vector_type(4), aligned(1)));
typedef int v4i_any4 __attribute__((ext_vector_type(4), aligned(4)));
typedef int v2i_any __attribute__((ext_vector_type(2), aligned(1)));

template <class T> struct Piece {      // as they lie in memory
  v4i raw;
  template <bool NT = false>
  __device__ __forceinline__ void load(const void *base, int64_t at, int count) {
    const uint16_t *src = reinterpret_cast<const uint16_t *>(base) + at;
    if (count >= 8) {
      if constexpr (NT) raw = __builtin_nontemporal_load(reinterpret_cast<const v4i_any *>(src));
      else raw = *reinterpret_cast<const v4i_any *>(src);
    } else {
      raw = v4i{0, 0, 0, 0};
      uint16_t *h = reinterpret_cast<uint16_t *>(&raw);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = e < count ? src[e] : (uint16_t)0;
    }
  }
  __device__ __forceinline__ void values(float (&f)[8]) const {
    const uint16_t *h = reinterpret_cast<const uint16_t *>(&raw);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = Elem<T>::to_float(h[e]);
  }
  __device__ __forceinline__ void round(const float (&f)[8]) { raw = round8<T, false>(f); }
  template <bool NT = false>
  __device__ __forceinline__ void store(void *base, int64_t at, int count) const {
    uint16_t *dst = reinterpret_cast<uint16_t *>(base) + at;
    if (count >= 8) {
      if constexpr (NT) __builtin_nontemporal_store(v4i_any(raw), reinterpret_cast<v4i_any *>(dst));
      else *reinterpret_cast<v4i_any *>(dst) = raw;
    } else {
      const uint16_t *h = reinterpret_cast<const uint16_t *>(&raw);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < count) dst[e] = h[e];
    }
  }
};
template <> struct Piece<F32> {
  v4i raw[2];
  template <bool NT = false>
  __device__ __forceinline__ void load(const void *base, int64_t at, int count) {
    const int *src = reinterpret_cast<const int *>(base) + at;
    if (count >= 8) {
      if constexpr (NT) {
        raw[0] = __builtin_nontemporal_load(reinterpret_cast<const v4i_any4 *>(src));
        raw[1] = __builtin_nontemporal_load(reinterpret_cast<const v4i_any4 *>(src + 4));
      } else {
        raw[0] = *reinterpret_cast<const v4i_any4 *>(src);
        raw[1] = *reinterpret_cast<const v4i_any4 *>(src + 4);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) raw[e >> 2][e & 3] = e < count ? src[e] : 0;
    }
  }
  __device__ __forceinline__ void values(float (&f)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = __builtin_bit_cast(float, (int)raw[e >> 2][e & 3]);
  }
};

}  // namespace cummhip
