// sample_place.h — where a logit lies on the axis of a row's bins, and its weight there
// (sample.hip). Plain C++, the same on host and device.
#pragma once
#include <math.h>

#ifdef __HIP__
#define SF_PLACE __host__ __device__ __attribute__((always_inline)) inline
#else
#define SF_PLACE inline
#endif

constexpr int kBins = 256;
constexpr double kDelta = 0.125;    // nats a bin

// 1 / (T kDelta): a logit's place on the bins' axis is x times it. The floor keeps an
// infinite temperature from turning infinite logits into NaN.
SF_PLACE double bins_per_logit(float T) { return fmax(1.0 / ((double)T * kDelta), 1e-300); }

// A logit's number on the axis: x per + kAxis, product and sum rounded each on its own,
// whatever the row's maximum. It is a multiple of 2^-33 everywhere: sums from 2^20 on are
// (of 2^-32), and a product below -2^19 is one and its sum exact. So a number's difference
// to a whole one is exact as far as the 4096 bins below it.
constexpr double kAxis = 1572864.0;  // 1.5 2^20
SF_PLACE double axis_of(float x, double per) {
#pragma clang fp contract(off)
  const double t = (double)x * per;
  return t + kAxis;
}
// That difference to the bin number `top` in 32 fractional bits: the sum with 1.5 2^20 holds
// the whole part in its high word and the rest in its low word. Its rounding (to even, of an
// exact value) commutes with a shift by whole numbers, so every chunk and the row agree on a
// logit's bin and weight.
SF_PLACE unsigned long long place_of(float x, double per, double top) {
#pragma clang fp contract(off)
  const double d = fmax(axis_of(x, per) - top, -4096.0) + 1572864.0;
  unsigned long long v;
  __builtin_memcpy(&v, &d, 8);
  return v;
}
SF_PLACE int whole_of(unsigned long long place) { return (int)(place >> 32 & 0xfffff) - 0x80000; }
// The bin number of a row's (chunk's) maximum: its own place relative to it is in [0, 1).
SF_PLACE double top_bin(float m, double per) {
  const double f = floor(axis_of(m, per));
  return f + (double)whole_of(place_of(m, per, f));
}
// The logit that lies `bins` below the bin number `top` (off by the rounding of its parts).
SF_PLACE double logit_at(double top, double bins, double per) { return (top - kAxis - bins) / per; }

struct Binned {
  int bin;  // below the bin of `top`; kBins and more: no weight
  unsigned long long w;
};
// Where x lies below the bin number `top`, and its weight (plus `add`). With s / 2^32 the
// place's distance from the bin's middle, y = kDelta s / 2^32 and 2^36 e^y = 2^36 + 2 s +
// 2^36 (y^2 / 2 + ... + y^5 / 120), the bracket in fp32: its rounding (0.002 2^-23) and the
// next term (y^6 / 720) are 3e-10 at most.
SF_PLACE Binned bin_of(float x, double per, double top, unsigned long long add = 0) {
  static_assert(kDelta == 0.125, "2^36 kDelta s / 2^32 = 2 s");
  const unsigned long long v = place_of(x, per, top);
  const int s = (int)((unsigned)v ^ 0x80000000u);
  const float y = (float)s * (float)(kDelta * 0x1p-32);
  const float tail = y * y * fmaf(y, fmaf(y, fmaf(y, 0x1p36f / 120, 0x1p36f / 24), 0x1p36f / 6), 0x1p35f);
  return Binned{-whole_of(v), (unsigned long long)((long long)s * 2 + (long long)((1ull << 36) + add)) + (unsigned)tail};
}
