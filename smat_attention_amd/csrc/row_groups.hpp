// Rows read and written eight values at a time, at the element's own alignment (a wide global
// access on gfx950 needs no more).
#pragma once

#include <type_traits>

#include "smat_common.hpp"

namespace smat {

// Eight consecutive values of a row as they come, at the element's own alignment.
template <typename In> struct Raw {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  typedef uint32_t u4h __attribute__((ext_vector_type(4), aligned(2)));
  typedef uint32_t u4f __attribute__((ext_vector_type(4), aligned(4)));
  typedef typename std::conditional<sizeof(In) == 2, u4h, u4f>::type u4u;
  static constexpr int N = sizeof(In) / 2;
  u4 x[N];
  __device__ __forceinline__ void load(const In* p) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = reinterpret_cast<const u4u*>(p)[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = u4{0, 0, 0, 0};
  }
  // Drops the first `by` values (0 <= by < 8): later ones move up, zeros follow.
  __device__ __forceinline__ void drop(int by) {
    uint32_t* d = reinterpret_cast<uint32_t*>(x);
    constexpr int W = 4 * N;
    if constexpr (sizeof(In) == 4) {
#pragma unroll
      for (int b = 4; b > 0; b >>= 1)
        if (by & b) {
#pragma unroll
          for (int i = 0; i < W; ++i) d[i] = i + b < W ? d[i + b] : 0;
        }
    } else {
#pragma unroll
      for (int b = 2; b > 0; b >>= 1)
        if (by & (2 * b)) {
#pragma unroll
          for (int i = 0; i < W; ++i) d[i] = i + b < W ? d[i + b] : 0;
        }
      if (by & 1) {
#pragma unroll
        for (int i = 0; i < W; ++i) d[i] = (d[i] >> 16) | (i + 1 < W ? d[i + 1] << 16 : 0);
      }
    }
  }
  __device__ __forceinline__ void values(f32x4& a, f32x4& b) const {
    if constexpr (__is_same(In, float)) {
      a = __builtin_bit_cast(f32x4, x[0]);
      b = __builtin_bit_cast(f32x4, x[1]);
    } else if constexpr (__is_same(In, bf16)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        a[2 * i] = __uint_as_float(x[0][i] << 16);
        a[2 * i + 1] = __uint_as_float(x[0][i] & 0xffff0000u);
        b[2 * i] = __uint_as_float(x[0][i + 2] << 16);
        b[2 * i + 1] = __uint_as_float(x[0][i + 2] & 0xffff0000u);
      }
    } else {
      const f16x8 h = __builtin_bit_cast(f16x8, x[0]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = (float)h[i];
        b[i] = (float)h[i + 4];
      }
    }
  }
};

// Eight values to p, rounded to Out; of them `nv` where the row ends before the eighth.
template <typename Out>
__device__ __forceinline__ void store8(Out* p, const f32x4& a, const f32x4& b, int nv) {
  if (nv >= 8) {
    if constexpr (sizeof(Out) == 2) {
      typedef Out out8u __attribute__((ext_vector_type(8), aligned(2)));
      out8u y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        y[i] = from_f32<Out>(a[i]);
        y[i + 4] = from_f32<Out>(b[i]);
      }
      *reinterpret_cast<out8u*>(p) = y;
    } else {
      typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
      reinterpret_cast<f32x4u*>(p)[0] = a;
      reinterpret_cast<f32x4u*>(p)[1] = b;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < nv) p[i] = from_f32<Out>(i < 4 ? a[i & 3] : b[i & 3]);
  }
}

}  // namespace smat
