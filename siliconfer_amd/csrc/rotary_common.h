// rotary_common.h — what the kernels that turn heads share: the angle's cosine and sine,
// positions given row by row, 16 bytes of a row as fp32 values.
#pragma once
#include <math.h>

#include "sf_common.h"

// The turned pair, products and sums rounded each on its own.
__device__ __forceinline__ float2_t turn(float x1, float x2, float2_t cs) {
#pragma clang fp contract(off)
  return float2_t{x1 * cs.x - x2 * cs.y, x2 * cs.x + x1 * cs.y};
}

// cos and sin of a: a less its nearest multiple of pi / 2 (in two parts, so that what is
// left is exact to 2^-53 of the angle), then the series of sine and cosine on [-pi/4, pi/4]
// in 64 bits, to r^11 and r^12: 7e-12 at most; LONG: to r^13 and r^14, 2e-14.
template <bool LONG>
__device__ __forceinline__ void rotary_sincos(double a, double &cos_a, double &sin_a) {
  const double n = rint(a * 0.63661977236758134308);
  const double r = fma(-n, 6.123233995736766036e-17, fma(-n, 1.57079632679489661923, a)), z = r * r;
  double s = -1.0 / 39916800, c = 1.0 / 479001600;
  if constexpr (LONG) {
    s = fma(1.0 / 6227020800, z, s);
    c = fma(-1.0 / 87178291200, z, c);
  }
  s = fma(s, z, 1.0 / 362880);
  c = fma(c, z, -1.0 / 3628800);
  s = fma(s, z, -1.0 / 5040);
  c = fma(c, z, 1.0 / 40320);
  s = fma(s, z, 1.0 / 120);
  c = fma(c, z, -1.0 / 720);
  s = fma(s, z, -1.0 / 6);
  c = fma(c, z, 1.0 / 24);
  s = fma(s * z, r, r);
  c = fma(fma(c, z, -0.5), z, 1.0);
  const int q = (int)((long long)n & 3);  // a = r + q pi / 2
  const double cq = q & 1 ? s : c, sq = q & 1 ? c : s;
  cos_a = q == 1 || q == 2 ? -cq : cq;
  sin_a = q & 2 ? -sq : sq;
}

// cos and sin of pos * f times scale, in fp32: the nearest fp32 values but for one in some
// thousands. Some 30 64-bit operations a pair (the library's sincos takes a longer
// reduction for far positions: 16 tokens near 500000 10.6 us, this 3.0).
__device__ __forceinline__ float2_t rotary_cs(long long pos, double f, float scale) {
  double c, s;
  rotary_sincos<false>((double)pos * f, c, s);
  return float2_t{(float)(scale * c), (float)(scale * s)};
}

// e / n by a product with ceil(2^32 / n), exact below 2^16; 0 stands for a division by 1.
__host__ __device__ inline uint32_t div_inv(int n) { return n == 1 ? 0 : (uint32_t)(((1ull << 32) + n - 1) / n); }
__device__ __forceinline__ int div_by(int e, uint32_t inv) { return inv ? (int)__umulhi((uint32_t)e, inv) : e; }

struct RotaryPos {
  const void *p;    // [B][T] or, stride_b = 0, [T]
  int i64;
  long long stride_b;
  __device__ __forceinline__ long long at(int b, int t) const {
    const size_t i = (size_t)b * stride_b + t;
    return i64 ? ((const long long *)p)[i] : (long long)((const int *)p)[i];
  }
};

// 16 bytes: 8 (4) values in fp32
template <int DT>
struct Vec {
  static constexpr int E = DT == SF_F32 ? 4 : 8;
  float v[E];
  __device__ __forceinline__ void load(u32x4 w) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = w[j];
      if constexpr (DT == SF_F32) {
        v[j] = sf_bitcast<float>(x);
      } else if constexpr (DT == SF_F16) {
        v[2 * j] = (float)sf_bitcast<f16>((uint16_t)(x & 0xffffu));
        v[2 * j + 1] = (float)sf_bitcast<f16>((uint16_t)(x >> 16));
      } else {
        v[2 * j] = sf_bitcast<float>(x << 16);
        v[2 * j + 1] = sf_bitcast<float>(x & 0xffff0000u);
      }
    }
  }
  __device__ __forceinline__ u32x4 pack() const {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == SF_F32) {
        w[j] = sf_bitcast<uint32_t>(v[j]);
      } else if constexpr (DT == SF_F16) {
        w[j] = sf_bitcast<uint16_t>((f16)sf_opaque(v[2 * j])) | (uint32_t)sf_bitcast<uint16_t>((f16)sf_opaque(v[2 * j + 1])) << 16;
      } else {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        w[j] = sf_bitcast<uint32_t>(__builtin_convertvector(float2_t{v[2 * j], v[2 * j + 1]}, bf16x2));
      }
    }
    return w;
  }
};
