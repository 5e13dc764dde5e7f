// attn_common.h — what the attention kernels over the int8 cache share: exact
// conversion of the codes to MFMA operands, and reductions over the four lanes that
// hold one query row of a 16x16 tile.
#pragma once
#include "sf_common.h"

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));

// 8 int8 codes (two dwords, byte order kept) -> 8 exact fp16 values: the
// offset-binary byte b + 128 in the low mantissa byte of fp16 1024, minus 1152.
__device__ __forceinline__ half8_t i8x8_to_h8(uint32_t lo, uint32_t hi) {
  const uint32_t a = lo ^ 0x80808080u, b = hi ^ 0x80808080u;
  const half2_t off = {(f16)-1152.f, (f16)-1152.f};
  const half2_t p0 = sf_bitcast<half2_t>(__builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) + off;
  const half2_t p1 = sf_bitcast<half2_t>(__builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) + off;
  const half2_t p2 = sf_bitcast<half2_t>(__builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) + off;
  const half2_t p3 = sf_bitcast<half2_t>(__builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) + off;
  return half8_t{p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
}

// max / sum of a value and its partners 16 and 32 lanes away (see sf_swap16_pair)
__device__ __forceinline__ float max_x16_x32(float v) {
  float2_t p = sf_swap16_pair(v);
  v = fmaxf(p.x, p.y);
  p = sf_swap32_pair(v);
  return fmaxf(p.x, p.y);
}
__device__ __forceinline__ float sum_x16_x32(float v) {
  float2_t p = sf_swap16_pair(v);
  v = p.x + p.y;
  p = sf_swap32_pair(v);
  return p.x + p.y;
}
