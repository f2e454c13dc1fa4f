// How numbers become codes of 8 bits by their largest magnitude (kv_8bit.cu: of a head; int8_gemm_sm100.cu: of a token).
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace {

constexpr float LEAST = 7.888609052210118e-31f;                    // 2^-100: keeps scales and their inverses normal numbers

// Eight numbers as they come: one or two 16-byte vectors
template <typename T> struct Raw8 {
  uint4 u[sizeof(T) / 2];
};
template <typename T> __device__ __forceinline__ Raw8<T> load8(const T* p, bool vec) {
  Raw8<T> r;
  if (vec) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = ldg_act(p + 8 / (sizeof(T) / 2) * i);
  } else {
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = p[i];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.u[i] = reinterpret_cast<const uint4*>(t)[i];
  }
  return r;
}
template <typename T> __device__ __forceinline__ void numbers_of(const Raw8<T>& r, float* f) {
  if constexpr (sizeof(T) == 2) {
    unpack8(r.u[0], f);
  } else {
    f[0] = __uint_as_float(r.u[0].x); f[1] = __uint_as_float(r.u[0].y); f[2] = __uint_as_float(r.u[0].z); f[3] = __uint_as_float(r.u[0].w);
    f[4] = __uint_as_float(r.u[1].x); f[5] = __uint_as_float(r.u[1].y); f[6] = __uint_as_float(r.u[1].z); f[7] = __uint_as_float(r.u[1].w);
  }
}
// The largest magnitude's bits: of fp32 numbers, or of bf16 ones in both halves (as whole numbers NaN is above infinity and that above the rest)
template <typename T> __device__ __forceinline__ uint32_t most_of(const Raw8<T>& r, uint32_t m) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
    const uint32_t w[4] = {r.u[i].x, r.u[i].y, r.u[i].z, r.u[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 2) m = __vmaxu2(m, w[j] & 0x7fff7fffu);
      else m = max(m, w[j] & 0x7fffffffu);
    }
  }
  return m;
}
// How numbers become codes, by their largest magnitude
template <bool INT8> struct Coder {
  float scale, f, y, as;                                           // scale NaN: codes are 0
  bool last;
  __device__ __forceinline__ explicit Coder(float largest) {
    if (!(largest <= 3.402823466e38f)) {                           // an infinity or NaN is among them
      scale = __uint_as_float(0x7fc00000u);
      f = y = as = 0.f;
      last = false;
      return;
    }
    const float a = fmaxf(largest, LEAST);
    const int e = (int)(__float_as_uint(a) >> 23) - 127;           // a = 1.m 2^e, -100 <= e <= 127
    if constexpr (INT8) {
      // 127 x / a, correctly rounded by Markstein's method (1990: an estimate of the quotient from the rounded reciprocal, and one correction by its exact remainder), so that a tie is a tie: x = a / 2
      // is 63.5 whatever 1 / a rounds to.  Both sides are divided by 128 and by a power of two near a, which keeps 127 x and 1 / a among the normal numbers.  127 x is exact for bf16 numbers; of fp32 ones it is
      // rounded once before, so that a code may be the neighbour's where the exact quotient is within 2^-23 of itself from a border.
      const float down = __uint_as_float((uint32_t)(127 - min(e, 126)) << 23);
      scale = a / 127.f;
      as = a * down;
      y = __frcp_rn(as);
      f = down * (127.f / 128.f);
      last = false;
    } else {
      const int s = e - 8 + ((__float_as_uint(a) & 0x7fffffu) > 0x600000u);            // 448 = 1.75 * 2^8
      scale = __uint_as_float((uint32_t)(127 + s) << 23);
      f = __uint_as_float((uint32_t)(127 - s) << 23);
      last = s == 120;
    }
  }
  __device__ __forceinline__ uint2 operator()(const float* x) const {
    uint32_t c[8];
    if constexpr (INT8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {                                // (the sum's lowest bits are the rounded number: as = 0 gives 0)
        const float n = x[i] * f, q = n * y;
        c[i] = __float_as_uint(fmaf(fmaf(fmaf(-as, q, n), y, q), 128.f, 12582912.f));
      }
      if (as == 0.f) return make_uint2(0u, 0u);
      return make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
                        __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 t = make_float2(x[2 * i] * f, x[2 * i + 1] * f);
        if (last) t = make_float2(fminf(fmaxf(t.x, -240.f), 240.f), fminf(fmaxf(t.y, -240.f), 240.f));   // (256 would read back as 2^128)
        c[i] = __nv_cvt_float2_to_fp8x2(t, __NV_SATFINITE, __NV_E4M3);
      }
      if (f == 0.f) return make_uint2(0u, 0u);
      return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
    }
  }
};

}  // namespace
