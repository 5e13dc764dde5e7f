// attn_q4.hip — attention over a KV cache held in 4 bits (gfx950).
//
// For Tq query rows a sequence (row t sees the first n - Tq + t + 1 of its n slots):
//   out = softmax(scale q K^T) V,  K = s c + m and V alike, (s, m) a group of g dims.
// A group's part of a score is s (q . c) + m sum(q), of an output sum(p s c) + sum(p m):
// the codes c go through the matrix units as they are, s and m join in fp32.
//
// The codes as MFMA operands: v_mfma_f32_16x16x32_f16 takes fp16's subnormals at their
// value, so a code in the low bits of a half is c 2^-24, and one four bits higher 16 c 2^-24:
// w & 0x000f000f and w & 0x00f000f0 of a word of eight codes are two operand registers (codes
// 0, 4 and 1, 5), the same of w >> 8 the others: five operations for eight codes. The other
// operand takes the same order and, for the odd pairs, a sixteenth.
//
// k_q4_split: one workgroup a (split, kv head and 16 of its rows, sequence); its four waves
// take 64-slot tiles. S^T = K q^T and O^T = V^T P^T with the query rows on the 16-wide side:
//   * row m of S^T's block h is slot 4 m + h of the tile, so lane l holds column l % 16 and the 16
//     neighbouring slots 16 (l / 16) .. of it, value (h, i) slot 4 i + h;
//   * V^T comes through LDS with ds_read_b64_tr_b4, which hands a lane one dim's codes of 16
//     slots: both B operands' order;
//   * q (fp32) and P as fp16 high and low parts, q brought to a largest magnitude of 2^13..2^14
//     by a power of two a row, P times the V scale under 2^15 likewise: what the low part drops is
//     below 2^-22 of the value and, where a row's weights span more, 2^-30 of the row's largest.
//     fp16 and bf16 queries are exact in the high part alone. (Without P's low part, a bf16 output of
//     four ragged sequences of up to 32767 slots takes 32.5 us, not 36.7: every weight off by up to
//     2^-11, some percent of the outputs rounded the other way.)
//   * codes less 8, with 8 s joined to m, keep the products' sums small: the matrix units cut what
//     they add to a sum, 2^-24 of it each time. For a bf16 output the codes stand as they are.
// Maxima, sums, m's part and the partials are fp32.
#include <math.h>

#include "attn_common.h"
#include "sf_common.h"
#include "split_merge.h"

int sf_q4_cache_check(int D, int g);  // kv_q4.hip

namespace {

constexpr int kQaThreads = 256;
constexpr int kQaWaves = kQaThreads / 64;
constexpr int kQaMaxSplits = 128;
constexpr int kQaMaxSlots = 0x7fffff00;

struct Q4Attn {
  const void *q;
  const uint8_t *kc, *vc;
  const uint32_t *kp, *vp;
  void *out;
  float *part_acc, *part_ml;
  const int *lengths;
  int qdt, odt, T, T_max, T_cap, Tq, H, KVH, D, g, n_splits, first;
  float qscale;
};

__device__ __forceinline__ int q4_len(const int *lengths, int T, int T_max, int b) {
  const long long n = (long long)(lengths ? lengths[b] : 0) + T;
  return n < 0 ? 0 : n > T_max ? T_max : (int)n;
}

// The power of two that takes a magnitude v to [2^13, 2^14) (1 for 0, and within the
// range of fp32's exponents).
__device__ __forceinline__ float q4_fit14(float v) {
  const int e = (int)(sf_bitcast<uint32_t>(v) >> 23 & 255);
  const int f = 127 + 13 + 127 - e;
  return v == 0.f ? 1.f : sf_bitcast<float>((uint32_t)(f < 1 ? 1 : f > 253 ? 253 : f) << 23);
}

// Eight codes as fp16 subnormals: codes 0, 4, 1, 5, 2, 6, 3, 7, times 2^-24, the pairs 1, 5 and
// 3, 7 times 16 more.
__device__ __forceinline__ half8_t q4_codes(uint32_t w) {
  const uint32_t x = w >> 8;
  const u32x4 r = {w & 0x000f000fu, w & 0x00f000f0u, x & 0x000f000fu, x & 0x00f000f0u};
  return sf_bitcast<half8_t>(r);
}

// The operations that lift a word's codes into the mantissas of 1024 and 64: held in registers
// (an instruction takes one literal), made once by a kernel.
struct Q4Magic {
  uint32_t a = 0x64006400u, b = 0x54005400u;
  __device__ __forceinline__ void hold() { asm volatile("" : "+v"(a), "+v"(b)); }
  __device__ __forceinline__ void lift(uint32_t w, half2_t (&p)[4]) const {
    const uint32_t x = w >> 8;
    p[0] = sf_bitcast<half2_t>((w & 0x000f000fu) | a);
    p[1] = sf_bitcast<half2_t>((w & 0x00f000f0u) | b);
    p[2] = sf_bitcast<half2_t>((x & 0x000f000fu) | a);
    p[3] = sf_bitcast<half2_t>((x & 0x00f000f0u) | b);
  }
};

// Eight codes less `less`, exact: pairs 0, 4; 1, 5; 2, 6; 3, 7.
template <int LESS>
__device__ __forceinline__ void q4_numbers(const Q4Magic &g, uint32_t w, half2_t (&p)[4]) {
  constexpr f16 a = (f16)(-1024.f - LESS), b = (f16)(-64.f - LESS);
  g.lift(w, p);
  p[0] += half2_t{a, a};
  p[1] += half2_t{b, b};
  p[2] += half2_t{a, a};
  p[3] += half2_t{b, b};
}

template <int LESS>
__device__ __forceinline__ half8_t q4_lifted(const Q4Magic &g, uint32_t w) {
  half2_t p[4];
  q4_numbers<LESS>(g, w, p);
  return half8_t{p[0].x, p[0].y, p[1].x, p[1].y, p[2].x, p[2].y, p[3].x, p[3].y};
}

__device__ __forceinline__ float q4_lo(uint32_t w) { return (float)sf_bitcast<f16>((uint16_t)(w & 0xffffu)); }
__device__ __forceinline__ float q4_hi(uint32_t w) { return (float)sf_bitcast<f16>((uint16_t)(w >> 16)); }

// Two fp32 values as a pair of fp16 high parts and one of what they leave.
__device__ __forceinline__ void q4_halves(float a, float b, uint32_t &hi, uint32_t &lo) {
  a = sf_opaque(a);
  b = sf_opaque(b);
  const f16 x = (f16)a, y = (f16)b;
  hi = sf_bitcast<uint16_t>(x) | (uint32_t)sf_bitcast<uint16_t>(y) << 16;
  lo = sf_bitcast<uint16_t>((f16)(a - (float)x)) | (uint32_t)sf_bitcast<uint16_t>((f16)(b - (float)y)) << 16;
}

// Workgroups of k_q4_split that a CU's registers hold without spilling (three at 128 dims in two groups
// with PK = 4 spill six registers: four ragged sequences of up to 32767 slots, bf16, 36.5 us, not 33.3; one
// 19.0, not 16.1). Only the form for any head (groups = 0) spills at one, where DP is 128: 95 with fp32
// queries, 56 with others (69 for bf16 outputs), 29 at DP = 256 with fp32 queries.
__host__ __device__ constexpr int q4_resident(int DP, int groups, int PK, bool QSPLIT) {
  return groups == 0 || DP > 128 ? 1
         : DP == 64              ? groups == 1 ? PK > 1 ? 4 : 3 : PK == 4 && !QSPLIT ? 4 : PK == 1 ? 2 : 3
         : groups == 1           ? QSPLIT && PK < 4 ? 2 : 3
         : groups == 2 || PK == 4 ? 2
                                  : 1;
}

// Columns: where a kv head has at most 8 (4) rows, PK = 2 (4) groups of 16 / PK columns hold the
// same rows, and a column takes only the values of a quarter's h (two, one of h = 0 .. 3): the
// softmax's work a tile is that of the rows there are. Each column is a softmax state of its
// own until the waves' states merge.
// A state's reference m stays until a score passes it by 8, so that most tiles need no maximum
// across lanes and no rescaling; the factor that takes p s to fp16's range stays likewise until
// a product passes 2^15, and grows where a reference that moves shrinks the products behind it.
// It is 2^110 at most: a weight, up to 2^8, stays finite times it beside a scale of 0.
// DP: the head's dims rounded up to 64, 128 or 256. NGT groups of 32 KSGT dims fill it
// exactly, or 0, 0: any head and groups. QSPLIT: q in two parts. SIGNED: codes less 8.
// Bound by vector instructions and the waits between them. Traced, with the merge launch, 32 / 8
// heads of 128: four ragged sequences of up to 32767 slots, bf16, groups of 64 (111 MB) 29.4 + 4.7
// us, the SIMDs issuing vector instructions 59% of the time of busy CUs (of some 690 a tile 290 turn
// codes into operands); one sequence of 131071, fp16, groups of 128 (143 MB) 30.9 + 4.5, 4.6 TB/s in
// the split; sixteen of up to 4001 with fp32 queries (51 MB) 20.8 + 3.9, q in two parts. The form for
// any head is far from that: 32767 slots of 9 / 3 heads of 80 (8.7 MB) 28 us a call in fp32, 16 / 4
// heads of 256 in groups of 64 (38 MB) 50.
template <bool QSPLIT, bool SIGNED, int DP, int NGT, int KSGT, int PK>
__global__ void __launch_bounds__(kQaThreads, q4_resident(DP, NGT, PK, QSPLIT))
k_q4_split(Q4Attn a) {
  constexpr bool ANY = NGT == 0;
  constexpr float kCode = SIGNED ? 1.f : 16777216.f;  // what an operand of K's codes is to be multiplied by
  constexpr int KS = DP / 32, DB = DP / 16, NGM = ANY ? 8 : NGT;
  constexpr int RP = 16 / PK, HV = 4 / PK, NV = 4 * HV;  // rows, h's and values of a column
  constexpr int PITCH = DP / 2 + 8;  // 16 neighbouring rows' 8 bytes fall on different banks
  constexpr int OP = DP + 4;
  constexpr int kTile = 64 * PITCH, kPar = 64 * NGM * 4;
  constexpr int kWave = kTile + 4 * kPar + (NGM > 1 ? 256 : 0), kO = 16 * OP * 4;
  __shared__ __attribute__((aligned(16))) uint8_t smem[kQaWaves * (kWave > kO ? kWave : kO) + 2 * kQaWaves * 16 * 4];
  const int D = ANY ? a.D : DP, NG = ANY ? a.D / a.g : NGT, GW = (ANY ? a.g : 32 * KSGT) / 8;
  const int KSG = ANY ? (GW + 3) / 4 : KSGT, nks = ANY ? NG * KSG : KS;
  const int G = a.H / a.KVH, R = a.Tq * G, nrb = PK > 1 ? 1 : (R + 15) / 16;
  const int split = blockIdx.x, kvh = blockIdx.y / nrb, rb = blockIdx.y - kvh * nrb, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane & 15, g = lane >> 4, nr = min(16, R - 16 * rb), pg = hl / RP, h0 = HV * pg;
  const int r = 16 * rb + hl % RP, qt = min(r, R - 1) / G, qh = min(r, R - 1) - qt * G;
  const size_t bk = (size_t)b * a.KVH + kvh, base = bk * a.T_cap;
  const int rowb = D / 2;
  // the word of codes that k-step ks takes of a slot (a group's words shared out over the four lanes)
  auto word = [&](int ks) {
    const int gi = ks / KSG, c = g * KSG + ks - gi * KSG;
    return c < GW ? gi * GW + c : -1;
  };

  uint32_t kr[4][KS];  // the codes of slots 4 hl + h
  u32x4 vr[DP / 32];   // 16 bytes of V codes each, slot-major
  uint32_t pr[2][NGM];
  Q4Magic magic;
  magic.hold();
  auto k_codes = [&](uint32_t w) { return SIGNED ? q4_lifted<8>(magic, w) : q4_codes(w); };
  // (slots are clamped into the cache; a tile's addresses are its own and a lane's 32-bit offset)
  auto load_k = [&](int j) {
    const uint8_t *const at = a.kc + (base + 64 * (size_t)j) * rowb;
    const int left = a.T_cap - 1 - 64 * j;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const uint32_t row = (uint32_t)(min(4 * hl + h, left) * rowb);
      if constexpr (!ANY) {
#pragma unroll
        for (int gi = 0; gi < NGT; ++gi) {
          const uint8_t *w = at + (row + 4 * KSGT * g + 16 * KSGT * gi);
          if constexpr (KSGT == 4) {
            const u32x4 x = *(const u32x4 *)w;
#pragma unroll
            for (int k = 0; k < 4; ++k) kr[h][gi * KSGT + k] = x[k];
          } else if constexpr (KSGT == 2) {
            const u32x2 x = *(const u32x2 *)w;
            kr[h][gi * KSGT] = x.x;
            kr[h][gi * KSGT + 1] = x.y;
          } else {
            kr[h][gi] = *(const uint32_t *)w;
          }
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if (ks >= nks) break;
          const int w = word(ks);
          kr[h][ks] = w >= 0 ? *(const uint32_t *)(at + (row + 4 * w)) : 0u;
        }
      }
    }
  };
  auto load_v = [&](int j) {
    const uint8_t *const at = a.vc + (base + 64 * (size_t)j) * rowb;
    const int left = a.T_cap - 1 - 64 * j;
    const int n16 = D / 32;  // 16-byte pieces a slot, and half a one where D is an odd multiple of 16
    if (!ANY || D % 32 == 0) {
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        if (ANY && i >= n16) break;
        const int e = lane + 64 * i, tok = e / n16, c = e - tok * n16;
        vr[i] = *(const u32x4 *)(at + (uint32_t)(min(tok, left) * rowb + 16 * c));
      }
    } else {
      const int n8 = D / 16;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        uint32_t x[4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int e = lane + 64 * (2 * i + u), tok = min(e / n8, 63), c = e - e / n8 * n8;
          const u32x2 w = *(const u32x2 *)(at + (uint32_t)(min(tok, left) * rowb + 8 * c));
          x[2 * u] = w.x;
          x[2 * u + 1] = w.y;
        }
        vr[i] = u32x4{x[0], x[1], x[2], x[3]};
      }
    }
  };
  auto load_p = [&](int j) {
    const size_t at = (base + 64 * (size_t)j) * NG;
    const int last = min(a.T_cap - 64 * j, 64) * NG - 1;  // (slots first: a capacity times its groups may pass 2^31)
#pragma unroll
    for (int i = 0; i < NGM; ++i) {
      if (ANY && i >= NG) break;
      const uint32_t e = (uint32_t)min(lane + 64 * i, last);
      pr[0][i] = (a.kp + at)[e];
      pr[1][i] = (a.vp + at)[e];
    }
  };

  const int n = q4_len(a.lengths, a.T, a.T_max, b);
  const int ntot = max(0, n - a.Tq + (16 * rb + nr - 1) / G + 1 + 63) / 64;  // up to the last row's own slot
  const int j0 = split + a.n_splits * wave, jstep = a.n_splits * kQaWaves;
  if (j0 < ntot) {
    load_k(j0);
    load_p(j0);
    load_v(j0);
  }
  const int lim = r < R ? max(0, n - a.Tq + qt + 1) : 0, lim_all = n - a.Tq + 16 * rb / G + 1;  // (of every row)

  // q in the codes' order, and its sum over each group (as the codes stand, times 2^-24)
  half8_t qh8[KS], ql8[QSPLIT ? KS : 1];
  float qs[NGM];
  float qmul;
  {
    float f[KS][8], top = 0.f;
    const size_t q0 = (((size_t)b * a.Tq + qt) * a.H + (size_t)kvh * G + qh) * D;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int w = ANY && ks >= nks ? -1 : word(ks);
      if (w >= 0) {
        if (a.qdt == SF_F32) sf_load8_as_f32<SF_F32>(a.q, q0 + 8 * w, f[ks]);
        else if (a.qdt == SF_F16) sf_load8_as_f32<SF_F16>(a.q, q0 + 8 * w, f[ks]);
        else sf_load8_as_f32<SF_BF16>(a.q, q0 + 8 * w, f[ks]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[ks][i] = r < R && w >= 0 ? f[ks][i] : 0.f;
        top = fmaxf(top, fabsf(f[ks][i]));
      }
    }
    const float up = q4_fit14(max_x16_x32(top));
    qmul = a.qscale == 0.f ? 1.f : fminf(fmaxf(fabsf(a.qscale) / up * kCode, 1.0e-37f), 1.0e36f);
    // (scores are compared before they are scaled: the scale's sign goes to q)
    const float by = a.qscale < 0.f ? -up : a.qscale > 0.f ? up : 0.f;
#pragma unroll
    for (int gi = 0; gi < NGM; ++gi) {
      float s = 0.f;
      if (!ANY || gi < NG) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          if (ks / KSG == gi)
#pragma unroll
            for (int i = 0; i < 8; ++i) s += f[ks][i] * by;
      }
      qs[gi] = sum_x16_x32(s) * (1.f / kCode);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = f[ks][(i >> 1) + 4 * (i & 1)] * by, part = !SIGNED && (i >> 1) & 1 ? 0.0625f : 1.f;
        const f16 hi = (f16)v;
        qh8[ks][i] = (f16)((float)hi * part);
        if constexpr (QSPLIT) ql8[ks][i] = (f16)((v - (float)hi) * part);
      }
  }

  uint8_t *const vt = smem + wave * kWave;
  // parameters a group, slot 16 g + 4 i + h at 16 h + 4 g + i: K's s and m (SIGNED: m + 8 s), V's alike
  float *const kss = (float *)(vt + kTile), *const kos = kss + 64 * NGM;
  float *const vss = kos + 64 * NGM, *const vos = vss + 64 * NGM;
  float *const vms = NGM > 1 ? vos + 64 * NGM : vss;  // a slot's largest V scale
  float m = -INFINITY, lsum = 0.f;  // base-2 softmax of the column
  float mul = 1.2980742e33f;        // 2^110 at most: the first tile sets it
  float am[NGM];                    // sum of p m (SIGNED: p (m + 8 s)) over the lane's slots
  float4_t O[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) O[d] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int gi = 0; gi < NGM; ++gi) am[gi] = 0.f;

  for (int j = j0; j < ntot; j += jstep) {
    const int tb = 64 * j;
    const bool more = j + jstep < ntot;
    // parameters and V codes into the wave's LDS; slots past the length stand for zeros
    if (tb + 64 > n) {
#pragma unroll
      for (int i = 0; i < NGM; ++i)
        if ((lane + 64 * i) / NG + tb >= n) pr[0][i] = pr[1][i] = 0u;
    }
#pragma unroll
    for (int i = 0; i < NGM; ++i) {
      if (ANY && i >= NG) break;
      const int e = lane + 64 * i, tok = e / NG, gi = e - tok * NG;
      const int to = 64 * gi + 16 * (tok & 3) + 4 * (tok >> 4) + (tok >> 2 & 3);
      kss[to] = q4_lo(pr[0][i]);
      kos[to] = SIGNED ? fmaf(8.f, q4_lo(pr[0][i]), q4_hi(pr[0][i])) : q4_hi(pr[0][i]);
      vss[to] = q4_lo(pr[1][i]);
      vos[to] = SIGNED ? fmaf(8.f, q4_lo(pr[1][i]), q4_hi(pr[1][i])) : q4_hi(pr[1][i]);
    }
    if (!ANY || D % 32 == 0) {
      const int n16 = D / 32;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        if (ANY && i >= n16) break;
        const int e = lane + 64 * i, tok = e / n16, c = e - tok * n16;
        uint2 *dst = (uint2 *)(vt + tok * PITCH + 16 * c);
        dst[0] = uint2{vr[i].x, vr[i].y};
        dst[1] = uint2{vr[i].z, vr[i].w};
      }
    } else {
      const int n8 = D / 16;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int e = lane + 64 * (2 * i + u), tok = e / n8, c = e - tok * n8;
          if (tok < 64) *(uint2 *)(vt + tok * PITCH + 8 * c) = uint2{vr[i][2 * u], vr[i][2 * u + 1]};
        }
    }
    if (more) {
      load_p(j + jstep);
      load_v(j + jstep);
    }
    if constexpr (NGM > 1) {
      float v = vss[lane];
#pragma unroll
      for (int gi = 1; gi < NGM; ++gi)
        if (!ANY || gi < NG) v = fmaxf(fabsf(v), fabsf(vss[64 * gi + lane]));
      vms[lane] = v;
    }
    float sc[NV];  // value 4 hh + i: slot tb + 16 g + 4 i + h0 + hh
#pragma unroll
    for (int e = 0; e < NV; ++e) sc[e] = 0.f;
#pragma unroll
    for (int gi = 0; gi < NGM; ++gi) {
      if (ANY && gi >= NG) break;
      float4_t S[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) S[h] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (ks / KSG != gi || ks >= nks) continue;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const half8_t x = k_codes(kr[h][ks]);
          S[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, qh8[ks], S[h], 0, 0, 0);
          if constexpr (QSPLIT) S[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ql8[ks], S[h], 0, 0, 0);
        }
      }
#pragma unroll
      for (int hh = 0; hh < HV; ++hh) {
        const float4_t ks = *(const float4_t *)(kss + 64 * gi + 16 * (h0 + hh) + 4 * g);
        const float4_t ko = *(const float4_t *)(kos + 64 * gi + 16 * (h0 + hh) + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = S[hh][i];
          if constexpr (PK == 2) x = pg ? S[2 + hh][i] : x;
          if constexpr (PK == 4) x = pg & 2 ? (pg & 1 ? S[3][i] : S[2][i]) : (pg & 1 ? S[1][i] : S[0][i]);
          sc[4 * hh + i] = fmaf(ks[i], x, fmaf(ko[i], qs[gi], sc[4 * hh + i]));
        }
      }
    }
    if (more) load_k(j + jstep);
    const bool masked = tb + 64 > lim_all;
    const int left = lim - tb - 16 * g - h0;  // the lane's slots 4 i + hh < left
    if (masked) {
#pragma unroll
      for (int e = 0; e < NV; ++e) sc[e] = 4 * (e & 3) + (e >> 2) < left ? sc[e] : -INFINITY;
    }
    float mx = sc[0];
#pragma unroll
    for (int e = 1; e < NV; ++e) mx = fmaxf(mx, sc[e]);
    mx *= qmul;
    float behind = 0.f;  // a bound of the products so far, where references move
    if (__any(mx > m + 8.f)) {
      const float M = max_x16_x32(mx), m_new = M > m + 8.f ? M : m;
      const float cf = __builtin_amdgcn_exp2f(m - sf_merge_mref(m_new));  // exp2(-inf) = 0
      behind = fmaxf(cf * (32768.f / mul), 6.3108872e-30f);  // (2^-97: a factor of 2^110)
      m = m_new;
      lsum *= cf;
#pragma unroll
      for (int gi = 0; gi < NGM; ++gi) am[gi] *= cf;
#pragma unroll
      for (int d = 0; d < DB; ++d) O[d] *= cf;
    }
    const float m_ref = sf_merge_mref(m);
    float pt = 0.f;
#pragma unroll
    for (int hh = 0; hh < HV; ++hh) {
      const float4_t v = *(const float4_t *)(vms + 16 * (h0 + hh) + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 4 * hh + i;
        sc[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], qmul, -m_ref));
        lsum += sc[e];
        pt = fmaxf(pt, fabsf(sc[e] * v[i]));  // (0 or NaN, which counts for nothing, past a row's end)
      }
    }
    if (__any(behind > 0.f || pt * mul > 32768.f)) {
      const float top = max_x16_x32(pt), was = mul;
      if (top * mul > 32768.f) mul = q4_fit14(top);
      else if (behind > 0.f) mul = fmaxf(mul, q4_fit14(fmaxf(top, behind)));
#pragma unroll
      for (int d = 0; d < DB; ++d) O[d] *= mul / was;
    }
    float pm[NV];
#pragma unroll
    for (int e = 0; e < NV; ++e) pm[e] = sc[e] * mul;
#pragma unroll
    for (int gi = 0; gi < NGM; ++gi) {
      if (ANY && gi >= NG) break;
      // P's operands: values (h, 0), (h, 1) of a register pair go with dword 0, (h, 2), (h, 3) with
      // dword 1; a column's registers of other h's hold zeros
      u32x4 ph[2], pl[2];
      float acc = am[gi];
#pragma unroll
      for (int hh = 0; hh < HV; ++hh) {
        float4_t vs = *(const float4_t *)(vss + 64 * gi + 16 * (h0 + hh) + 4 * g);
        float4_t vo = *(const float4_t *)(vos + 64 * gi + 16 * (h0 + hh) + 4 * g);
        if (masked) {  // what lies past a row's end weighs exactly 0, whatever its parameters hold
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            vs[i] = 4 * i + hh < left ? vs[i] : 0.f;
            vo[i] = 4 * i + hh < left ? vo[i] : 0.f;
          }
        }
        float pv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc = fmaf(vo[i], sc[4 * hh + i], acc);
          pv[i] = vs[i] * pm[4 * hh + i];
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t x, y;
          q4_halves(pv[2 * w], pv[2 * w + 1], x, y);
#pragma unroll
          for (int p = 0; p < PK; ++p) {
            ph[w][HV * p + hh] = PK == 1 || pg == p ? x : 0u;
            pl[w][HV * p + hh] = PK == 1 || pg == p ? y : 0u;
          }
        }
      }
      am[gi] = acc;
      typedef int v2i __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        if (ANY ? 16 * d < gi * a.g || 16 * d >= (gi + 1) * a.g : d / (2 * (KSGT ? KSGT : 1)) != gi) continue;
        const v2i vw = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
            (__attribute__((address_space(3))) v2i *)(vt + (16 * g + hl) * PITCH + 8 * d));
        const half8_t x0 = q4_lifted<SIGNED ? 8 : 0>(magic, (uint32_t)vw.x), x1 = q4_lifted<SIGNED ? 8 : 0>(magic, (uint32_t)vw.y);
        O[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x0, sf_bitcast<half8_t>(ph[0]), O[d], 0, 0, 0);
        O[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x1, sf_bitcast<half8_t>(ph[1]), O[d], 0, 0, 0);
        O[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x0, sf_bitcast<half8_t>(pl[0]), O[d], 0, 0, 0);
        O[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x1, sf_bitcast<half8_t>(pl[1]), O[d], 0, 0, 0);
      }
    }
  }
  lsum = sum_x16_x32(lsum);
#pragma unroll
  for (int gi = 0; gi < NGM; ++gi) am[gi] = sum_x16_x32(am[gi]);

  // merge the waves' and columns' states through LDS into the split's partial, or the output
  __syncthreads();
  float *os = (float *)smem;  // [wave][16][OP]
  float *ms = (float *)(smem + kQaWaves * (kWave > kO ? kWave : kO)), *ls = ms + kQaWaves * 16;
  if (g == 0) {
    ms[wave * 16 + hl] = m;
    ls[wave * 16 + hl] = lsum;
  }
  const float un = 1.f / mul;
#pragma unroll
  for (int d = 0; d < DB; ++d) {
    if (ANY && 16 * d >= D) break;
    float add = am[0];
#pragma unroll
    for (int gi = 1; gi < NGM; ++gi)
      if (ANY ? 16 * d / a.g == gi : d / (2 * (KSGT ? KSGT : 1)) == gi) add = am[gi];
    *(float4_t *)(os + (wave * 16 + hl) * OP + 16 * d + 4 * g) = O[d] * un + add;
  }
  __syncthreads();
  const int nq = D / 4;
  for (int e = tid; e < nr * nq; e += kQaThreads) {
    const int rr = e / nq, d4 = (e - rr * nq) * 4;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kQaWaves * PK; ++w) M = fmaxf(M, ms[w * RP + rr]);
    const float M_ref = sf_merge_mref(M);
    float L = 0.f;
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kQaWaves * PK; ++w) {
      const float wt = sf_merge_weight(ms[w * RP + rr], M_ref);
      L = fmaf(wt, ls[w * RP + rr], L);
      acc += *(const float4_t *)(os + (w * RP + rr) * OP + d4) * wt;
    }
    if (a.n_splits > 1) {
      const size_t row = (bk * R + 16 * rb + rr) * a.n_splits + split;
      *(float4_t *)(a.part_acc + row * D + d4) = acc;
      if (d4 == 0) *(float2_t *)(a.part_ml + row * 2) = float2_t{M, L};
    } else {
      const int ro = 16 * rb + rr, t = ro / G, hh = kvh * G + ro - t * G;
      const size_t o = (((size_t)b * a.Tq + t) * a.H + hh) * D + d4;
#pragma unroll
      for (int i = 0; i < 4; ++i) sf_store_dt(a.out, a.odt, o + i, sf_merge_finish(L, acc[i]));
    }
  }
}

// The second launch: a workgroup merges one query row's partials, every thread four dims of
// some of the splits, the parts then summed in LDS, all loads of a thread in flight at once.
__global__ void __launch_bounds__(kQaThreads)
k_q4_merge(const float *__restrict__ part_acc, const float *__restrict__ part_ml, void *__restrict__ out, int odt, int Tq,
           int H, int KVH, int D, int S) {
  constexpr int kPre = 4;
  __shared__ __attribute__((aligned(16))) float sm[kQaMaxSplits + 4 * kQaThreads];
  const int row = blockIdx.x, nq = D / 4, parts = kQaThreads / nq, q = threadIdx.x % nq, part = threadIdx.x / nq;
  const int lane = threadIdx.x & 63;
  const float2_t *ml = (const float2_t *)part_ml + (size_t)row * S;
  const float4_t *acc = (const float4_t *)part_acc + (size_t)row * S * nq + q;
  const float2_t e0 = ml[min(lane, S - 1)], e1 = ml[min(lane + 64, S - 1)];
  float4_t pre[kPre];
#pragma unroll
  for (int k = 0; k < kPre; ++k) pre[k] = acc[(size_t)min(part + k * parts, S - 1) * nq];
  const float m0 = lane < S ? e0.x : -INFINITY, m1 = lane + 64 < S ? e1.x : -INFINITY;
  const float M = sf_merge_mref(sf_wave_max(fmaxf(m0, m1)));
  const float w0 = sf_merge_weight(m0, M), w1 = sf_merge_weight(m1, M);
  const float L = sf_wave_sum((lane < S ? w0 * e0.y : 0.f) + (lane + 64 < S ? w1 * e1.y : 0.f));
  float *w = sm;
  float4_t *p = (float4_t *)(sm + kQaMaxSplits);  // [parts][nq]
  if (threadIdx.x < 64) {
    w[lane] = w0;
    w[lane + 64] = w1;
  }
  __syncthreads();
  float4_t v = {0.f, 0.f, 0.f, 0.f};
  if (part < parts) {
#pragma unroll
    for (int k = 0; k < kPre; ++k)
      if (part + k * parts < S) v += pre[k] * w[part + k * parts];
    for (int s = part + kPre * parts; s < S; s += parts) v += acc[(size_t)s * nq] * w[s];
    p[part * nq + q] = v;
  }
  __syncthreads();
  if (part == 0) {
    for (int i = 1; i < parts; ++i) v += p[i * nq + q];
    const int G = H / KVH, R = Tq * G, bk = row / R, r = row - bk * R;
    const int b = bk / KVH, t = r / G, h = (bk - b * KVH) * G + r - t * G;
    const size_t o = (((size_t)b * Tq + t) * H + h) * D + 4 * q;
#pragma unroll
    for (int i = 0; i < 4; ++i) sf_store_dt(out, odt, o + i, sf_merge_finish(L, v[i]));
  }
}

// ---------------------------------------------------------------------------
// many rows: prompts
// ---------------------------------------------------------------------------
// Two launches. k_q4_spread takes the cache's values m + s c once for all rows, as fp16 (SPLIT:
// and what that leaves, a second fp16), into the workspace in the order of the matrix
// operands, 1 KB a fragment, blocks of 32 slots:
//   * K: a lane makes its slot's fragments from neighbouring words of codes, q is loaded in
//     the same order of dims;
//   * V: codes through LDS and ds_read_b64_tr_b4, a lane then holds one dim's codes of 16
//     slots in the order in which S^T leaves the weights in registers.
// k_q4_rows: a workgroup owns 128 consecutive (row, head) columns c = t G + h of one kv head,
// 32 a wave, and walks the tiles (64 slots; SPLIT: 32) up to its last row's own slot. KG = 2:
// two at a time, waves 0..3 the even ones, waves 4..7 the odd ones, whose states merge at the
// end. A tile goes straight to LDS, the next one while it is worked on: S^T = K q^T, a base-2
// softmax a column and O^T = V^T P^T on v_mfma_f32_32x32x16_f16, the next tile's scores
// between the softmax's instructions.
// For a bf16 output of 16-bit queries P and the values are rounded to fp16, 2^-11 of each at most: P's
// and V's rounding move an output by that much of sum(p |v|), an eighth of what its own (2^-8) may.
// K's is multiplied by the score's size in the exponent: a weight is off by up to 2^-11 of
// scale sum |q k|, what a K held in fp16 would give. (K in two parts: 1500 rows below 74 us instead of
// 52, 4096 rows 242 instead of 180.) Other outputs, and fp32 queries, take three products
// of the high and low parts.
// What fp16 cannot hold: a tile of K, and a group of a tile of V, that has values past 65504 is taken
// at 2^-6 (K's scores and V's sums times 2^6 again; what it holds beside them is off by 2^-15 at
// most: s and m by 2^-19 each); parameters that are not finite stand as zeros in V, and the columns
// that see them get NaN in their group's dims.
// Measured, 32 / 8 heads of 128, bf16: 4096 rows 168 us (818 TFLOP/s of the products; a large
// fp16 matrix product reaches 1215 on this card), 1500 rows behind 300 51.6 us, of which 6 the
// first launch; both bound by the softmax's instructions and the products beside them, the
// second also by the longest columns' 28 tiles one after the other. (Made within one kernel,
// each workgroup its tiles' values through LDS and two barriers a tile: 203 and 58.)

// The workspace: blocks [B KVH][blocks of 32 slots][part][K fragments, V fragments], then
// flags [B KVH][tiles of 64][2].
__host__ __device__ constexpr size_t q4_block_bytes(int D, int parts) { return (size_t)parts * D / 8 * 1024; }
__host__ __device__ inline size_t q4_tiles(int T_max) { return ((size_t)T_max + 63) / 64; }

// Whether a parameter word is not finite, or stands for values past fp16's range (the last
// code's; m itself is fp16).
__device__ __forceinline__ bool q4_none(uint32_t w) { return (w & 0x7fffu) >= 0x7c00u || (w >> 16 & 0x7fffu) >= 0x7c00u; }
__device__ __forceinline__ bool q4_past(uint32_t w) { return !q4_none(w) && fabsf(fmaf(15.f, q4_lo(w), q4_hi(w))) >= 65520.f; }
// A tile's flags of V: a bit a group that is taken at 2^-6, and
constexpr uint32_t kV6 = 15, kVNone = 256;  // something not finite

// One workgroup a tile of 64 slots of one kv head.
template <bool SPLIT, int D>
__global__ void __launch_bounds__(256)
k_q4_spread(Q4Attn a, uint8_t *__restrict__ ws, uint32_t *__restrict__ flags) {
  constexpr int NFW = D / 32;      // K fragments a wave makes of its 32 slots, of 2 NFW
  constexpr int NDB = D / 32;      // 32-dim blocks
  constexpr int PARTS = SPLIT ? 2 : 1, PITCH = D / 2 + 8;
  typedef uint32_t Words __attribute__((ext_vector_type(NFW)));  // 16 (8) bytes of codes
  __shared__ __attribute__((aligned(16))) uint8_t raw[64 * PITCH];
  __shared__ __attribute__((aligned(16))) f16 vsm[2][NDB][64];  // s and m a group, in the order of the weights
  __shared__ uint32_t flag[2];
  const int j = blockIdx.x, bk = blockIdx.y, b = bk / a.KVH, NG = D / a.g;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = q4_len(a.lengths, a.T, a.T_max, b);
  if (64 * j >= n) return;
  const int tb = wave >> 1, w2 = wave & 1;          // K: the slots 32 tb + l32, fragments NFW w2 ..
  const int kword = 2 * NFW * w2 + NFW * h, kg = 8 * kword / a.g, krow = 32 * tb + l32;
  const int vtok = tid >> 2, vpiece = tid & 3;      // V: 16 (8) bytes of a slot
  const int ptok = tid / NG, pg = tid - ptok * NG;  // V: a slot's parameters of a group
  const bool has_p = tid < 64 * NG;
  const size_t at = (size_t)bk * a.T_cap + 64 * (size_t)j;
  const int left = a.T_cap - 1 - 64 * j, kt = min(krow, left);  // (slots are clamped into the cache)
  const Words kr = *(const Words *)(a.kc + at * (D / 2) + (uint32_t)(kt * (D / 2) + 4 * kword));
  const Words vr = *(const Words *)(a.vc + at * (D / 2) + (uint32_t)(min(vtok, left) * (D / 2) + 4 * NFW * vpiece));
  uint32_t kpr = (a.kp + at * NG)[(uint32_t)(kt * NG + kg)], vpr = 0;
  if (has_p) vpr = (a.vp + at * NG)[(uint32_t)(min(ptok, left) * NG + pg)];
  if (64 * j + krow >= n) kpr = 0;  // slots past the length stand for zeros
  if (64 * j + ptok >= n) vpr = 0;
  if (tid < 2) flag[tid] = 0;
  __syncthreads();
  const bool none = q4_none(vpr);
  if (q4_past(kpr)) atomicOr(&flag[0], 1u);
  if (q4_past(vpr)) atomicOr(&flag[1], 1u << pg);
  if (none) atomicOr(&flag[1], kVNone);
  uint2 *dst = (uint2 *)(raw + vtok * PITCH + 4 * NFW * vpiece);  // (rows on 8 bytes)
#pragma unroll
  for (int i = 0; i < NFW; i += 2) dst[i / 2] = uint2{vr[i], vr[i + 1]};
  __syncthreads();
  const uint32_t fk = flag[0], fv = flag[1];
  if (tid < 2) flags[((size_t)bk * q4_tiles(a.T_max) + j) * 2 + tid] = flag[tid];
  const float kdown = fk ? 0.015625f : 1.f, vdown = fv >> pg & 1 & kV6 ? 0.015625f : 1.f;
  Q4Magic magic;
  magic.hold();
  // eight values of one slot, or of eight slots (s, m one each), as operand parts
  auto values = [&](uint32_t w, const half2_t (&s)[4], const half2_t (&m)[4], half8_t &hi, half8_t &lo) {
    half2_t c8[4];
    q4_numbers<0>(magic, w, c8);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const half2_t v = __builtin_elementwise_fma(c8[p], s[p], m[p]);
      hi[2 * p] = v.x;
      hi[2 * p + 1] = v.y;
      if constexpr (SPLIT) {
        lo[2 * p] = (f16)(fmaf((float)c8[p].x, (float)s[p].x, (float)m[p].x) - (float)v.x);
        lo[2 * p + 1] = (f16)(fmaf((float)c8[p].y, (float)s[p].y, (float)m[p].y) - (float)v.y);
      }
    }
  };
  // fragment i of K (2 NFW a block) or V (2 NDB, after them) of block t
  uint8_t *const blocks = ws + ((size_t)bk * q4_tiles(a.T_max) + j) * 2 * q4_block_bytes(D, PARTS);
  auto put = [&](int t, int i, const half8_t &hi, const half8_t &lo) {
    half8_t *o = (half8_t *)(blocks + t * q4_block_bytes(D, PARTS)) + i * 64 + lane;
    o[0] = hi;
    if constexpr (SPLIT) o[4 * NFW * 64] = lo;
  };
  {
    f16 s = (f16)(q4_lo(kpr) * kdown), m = (f16)(q4_hi(kpr) * kdown);
    const half2_t s2 = {s, s}, m2 = {m, m}, sp[4] = {s2, s2, s2, s2}, mp[4] = {m2, m2, m2, m2};
#pragma unroll
    for (int i = 0; i < NFW; ++i) {
      half8_t hi, lo;
      values(kr[i], sp, mp, hi, lo);
      put(tb, NFW * w2 + i, hi, lo);
    }
  }
  if (has_p) {
    const int u = ptok & 31, e = 4 * (u >> 3) + (u & 3);
    const int to = 32 * (ptok >> 5) + 16 * (e >> 3) + 8 * (u >> 2 & 1) + (e & 7);
    vsm[0][pg][to] = none ? (f16)0.f : (f16)(q4_lo(vpr) * vdown);
    vsm[1][pg][to] = none ? (f16)0.f : (f16)(q4_hi(vpr) * vdown);
  }
  __syncthreads();
  constexpr int NR = D == 128 ? 2 : 1;  // transposing reads, two fragments each
  const int db = D == 128 ? wave : wave & 1, r0 = D == 128 ? 0 : wave >> 1, vg = 32 * db / a.g;
  typedef int v2i __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int jl = lane & 15, s0 = 2 * (r0 + r), jj = jl & 7, s = s0 + (jl >> 3);
    const int e = 8 * (s & 1) + (jj < 4 ? 2 * jj : 2 * (jj - 4) + 1);
    const int row = 32 * (s >> 1) + 8 * (e >> 2) + 4 * h + (e & 3);
    const v2i w = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
        (__attribute__((address_space(3))) v2i *)(raw + row * PITCH + 16 * db + 8 * (lane >> 4 & 1)));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const half8_t s8 = *(const half8_t *)&vsm[0][vg][16 * (s0 + i) + 8 * h];
      const half8_t m8 = *(const half8_t *)&vsm[1][vg][16 * (s0 + i) + 8 * h];
      const half2_t sp[4] = {{s8[0], s8[1]}, {s8[2], s8[3]}, {s8[4], s8[5]}, {s8[6], s8[7]}};
      const half2_t mp[4] = {{m8[0], m8[1]}, {m8[2], m8[3]}, {m8[4], m8[5]}, {m8[6], m8[7]}};
      half8_t hi, lo;
      values((uint32_t)(i ? w.y : w.x), sp, mp, hi, lo);
      put((s0 + i) >> 1, 2 * NFW + ((s0 + i) & 1) * NDB + db, hi, lo);
    }
  }
}

template <int QDT, bool SPLIT, int D, int KG>
__global__ void __launch_bounds__(256 * KG, 2)
k_q4_rows(Q4Attn a, const uint8_t *__restrict__ ws, const uint32_t *__restrict__ flags) {
  constexpr int NFW = D / 32, NDB = D / 32;
  constexpr int PARTS = SPLIT ? 2 : 1, QP = QDT == SF_F32 ? 2 : 1;
  static_assert(SPLIT || QDT != SF_F32, "fp32 queries keep both parts");
  constexpr int NT = SPLIT ? 1 : 2, TS = 32 * NT;  // blocks and slots a tile
  constexpr int BLOCK = (int)q4_block_bytes(D, PARTS), KB_ = 2 * NFW;  // V's fragments come after K's
  typedef float float16_t __attribute__((ext_vector_type(16)));
  constexpr int kTiles = 2 * KG * NT * BLOCK, kMerge = KG == 1 ? 0 : 4 * 64 * (16 * NDB + 2) * 4;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kTiles > kMerge ? kTiles : kMerge];  // [half][two in turn][tile]
  const int G = a.H / a.KVH, NG = D / a.g, ncol = a.Tq * G, ncb = (ncol + 127) / 128;
  // The heads of all sequences side by side, the longest columns first; where all workgroups
  // are resident at once, two on some CUs, the second of a CU comes to the shortest of the first.
  const int BK = a.n_splits, bk = (int)(blockIdx.x % (unsigned)BK), at = (int)(blockIdx.x / (unsigned)BK);
  const int c0 = (ncb - 1 - (at < a.first ? a.first - 1 - at : at)) * 128;
  const int b = bk / a.KVH, kvh = bk - b * a.KVH;
  const int tid = threadIdx.x & 255, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kgrp = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int n = q4_len(a.lengths, a.T, a.T_max, b);
  auto limit = [&](int c) { return max(0, n - a.Tq + c / G + 1); };  // slots column c sees
  const int cw = c0 + 32 * wave, c = min(cw + l32, ncol - 1);
  const int lim = limit(c), lo_lim = limit(min(cw, ncol - 1));
  const int hi_lim = cw < ncol ? limit(min(cw + 31, ncol - 1)) : 0;  // and the wave's
  const int ntot = (limit(min(c0 + 127, ncol - 1)) + TS - 1) / TS;
  const size_t qrow = ((size_t)b * a.Tq + c / G) * a.H + (size_t)kvh * G + c % G;

  const uint8_t *const src = ws + (size_t)bk * q4_tiles(a.T_max) * 2 * BLOCK;
  const uint32_t *const fl = flags + (size_t)bk * q4_tiles(a.T_max) * 2;
  uint8_t *const mine = lds + kgrp * 2 * NT * BLOCK;
  // Half a tile of the wave's own run of tiles (K's or V's fragments) to a buffer: 1 KB an
  // instruction, the four waves in turn.
  constexpr int HALF = BLOCK / PARTS / 2;  // bytes of K's, or V's, fragments of a block's part
  auto load = [&](int it, bool v) {
    const int j = KG * it + kgrp;
    if (j >= ntot) return;
#pragma unroll
    for (int i = 0; i < NT * PARTS * HALF / 4096; ++i) {
      const int u = 4 * i + wave, blk = u / (HALF / 1024), o = blk * 2 * HALF + (v ? HALF : 0) + u % (HALF / 1024) * 1024;
      __builtin_amdgcn_global_load_lds(
          (__attribute__((address_space(1))) void *)(src + (size_t)j * (NT * BLOCK) + o + 16 * lane),
          (__attribute__((address_space(3))) void *)(mine + (it & 1) * NT * BLOCK + o), 16, 0, 0);
    }
  };
  load(0, false);
  load(0, true);

  half8_t qf[QP][2 * NFW];
  float qmul;
  {
    float f[2 * NFW][8], top = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * NFW; ++i) {
      sf_load8_as_f32<QDT>(a.q, qrow * D + 8 * (2 * NFW * (i / NFW) + NFW * h + i % NFW), f[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(f[i][e]));
    }
    const float2_t tp = sf_swap32_pair(top);
    const float up = q4_fit14(fmaxf(tp.x, tp.y));
    qmul = a.qscale == 0.f ? 1.f : fminf(fmaxf(fabsf(a.qscale) / up, 1.0e-37f), 1.0e36f);
    // (scores are compared before they are scaled: the scale's sign goes to q)
    const float by = a.qscale < 0.f ? -up : a.qscale > 0.f ? up : 0.f;
#pragma unroll
    for (int i = 0; i < 2 * NFW; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // the codes' order: 0, 4, 1, 5, ..
        const float x = f[i][e] * by, y = f[i][e + 4] * by;
        if constexpr (QDT != SF_F32) {  // exact
          const auto w = __builtin_amdgcn_cvt_pkrtz(x, y);
          qf[0][i][2 * e] = (f16)w[0];
          qf[0][i][2 * e + 1] = (f16)w[1];
        } else {
          qf[0][i][2 * e] = (f16)x;
          qf[0][i][2 * e + 1] = (f16)y;
          qf[1][i][2 * e] = (f16)(x - (float)qf[0][i][2 * e]);
          qf[1][i][2 * e + 1] = (f16)(y - (float)qf[0][i][2 * e + 1]);
        }
      }
  }

  // Weights are 2^(score - m + 6), m a score that the row's largest passes by 8 at most: O is
  // rescaled when it would be more (with 32 columns a wave some maximum moves in most tiles),
  // the weights stay under fp16's end, and their low parts normal numbers down to 2^-20.
  constexpr float kP = 6.f, kSlack = 8.f;
  float m = -INFINITY, lsum = 0.f;
  float16_t O[NDB];
#pragma unroll
  for (int d = 0; d < NDB; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) O[d][e] = 0.f;

  // A tile's scores are made while the softmax of the one before runs: products and vector
  // instructions of one wave side by side.
  auto frag = [&](int it, int p, int t, int i) {
    return ((const half8_t *)(mine + (it & 1) * NT * BLOCK) + lane)[(t * BLOCK + p * (BLOCK / PARTS) + i * 1024) / 16];
  };
  auto score = [&](int it, int f0, int f1, float16_t (&S)[NT]) {  // k-steps f0 .. f1 of all blocks
#pragma unroll
    for (int f = f0; f < f1; ++f)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const half8_t x = frag(it, 0, t, f);
        if (f == 0) {
#pragma unroll
          for (int e = 0; e < 16; ++e) S[t][e] = 0.f;
        }
        S[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qf[0][f], S[t], 0, 0, 0);
        if constexpr (QP == 2) S[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qf[1][f], S[t], 0, 0, 0);
        if constexpr (SPLIT) S[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(frag(it, 1, t, f), qf[0][f], S[t], 0, 0, 0);
      }
  };
  auto step = [&](int it, float16_t (&S)[NT], float16_t (&next)[NT]) {
    const int j = KG * it + kgrp;
    __builtin_amdgcn_s_waitcnt((15 << 8) | (7 << 4));  // vmcnt(0): the wave's share of this V and the next K is in LDS
    __syncthreads();                                    // and the other waves'; the last V and this K are read
    load(it + 2, false);
    load(it + 1, true);
    if (TS * j >= hi_lim || j >= ntot) return;  // no column of the wave sees it (uniform)
    const uint32_t fk = fl[2 * (NT * j / 2)], fv = fl[2 * (NT * j / 2) + 1];
    const float mul = fk ? qmul * 64.f : qmul;
    if (TS * j + TS > lo_lim) {  // the lane's slots 32 t + 8 (e / 4) + 4 h + e % 4
      const int left = lim - TS * j - 4 * h;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) S[t][e] = 32 * t + 8 * (e >> 2) + (e & 3) < left ? S[t][e] : -INFINITY;
    }
    score(it + 1, 0, NFW, next);  // (past the last tile: whatever lies there, never used)
    float mx = S[0][0];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, S[t][e]);
    const float2_t mp = sf_swap32_pair(mx);
    const float m_new = fmaxf(m, fmaxf(mp.x, mp.y) * mul);
    if (__any(m_new > m + kSlack)) {
      const float cf = __builtin_amdgcn_exp2f(m - sf_merge_mref(m_new));  // exp2(-inf) = 0
      lsum *= cf;
#pragma unroll
      for (int d = 0; d < NDB; ++d) O[d] *= cf;
      m = m_new;
    }
    if (fv & kV6) {
#pragma unroll
      for (int d = 0; d < NDB; ++d) O[d] *= fv >> 32 * d / a.g & 1 ? 0.015625f : 1.f;
    }
    const float shift = kP - sf_merge_mref(m);
    score(it + 1, NFW, 2 * NFW, next);
    u32x4 ph[2 * NT], pl[2 * NT];
#pragma unroll
    for (int s = 0; s < 2 * NT; ++s)
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float x = __builtin_amdgcn_exp2f(fmaf(S[s >> 1][8 * (s & 1) + 2 * p], mul, shift));
        const float z = __builtin_amdgcn_exp2f(fmaf(S[s >> 1][8 * (s & 1) + 2 * p + 1], mul, shift));
        if constexpr (SPLIT) {
          lsum += x + z;
          uint32_t hi, lo;
          q4_halves(x, z, hi, lo);
          ph[s][p] = hi;
          pl[s][p] = lo;
        } else {  // rounded to fp16; their sum is the rounded weights', so that both are off alike
          const half2_t w = __builtin_convertvector(float2_t{x, z}, half2_t);
          ph[s][p] = sf_bitcast<uint32_t>(w);
          lsum = __builtin_amdgcn_fdot2(w, half2_t{(f16)1.f, (f16)1.f}, lsum, false);
        }
      }
    // (one product to some vector instructions, operands read ahead)
    constexpr int kProducts = NFW * NT * (SPLIT ? QP + 1 : 1), kVector = (SPLIT ? 9 : 4) * 16 * NT / kProducts;
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < kProducts; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, kVector / 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x400, 16 * NT / kProducts, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, kVector / 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    // fragments are read a batch ahead of the products that take them, two batches in turn;
    // neighbouring products belong to different sums
    constexpr int VB = SPLIT ? 2 : 4, NVB = 2 * NT * NDB / VB;
    half8_t y[2][PARTS][VB];
    auto fetch_v = [&](int bi) {
#pragma unroll
      for (int i = 0; i < VB; ++i)
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          const int s = (bi * VB + i) / NDB, d = (bi * VB + i) % NDB;
          y[bi & 1][p][i] = frag(it, p, s >> 1, KB_ + (s & 1) * NDB + d);
        }
    };
    fetch_v(0);
#pragma unroll
    for (int bi = 0; bi < NVB; ++bi) {
      if (bi + 1 < NVB) fetch_v(bi + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < VB; ++i) {
        const int s = (bi * VB + i) / NDB, d = (bi * VB + i) % NDB;
        const half8_t p = sf_bitcast<half8_t>(ph[s]);
        O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y[bi & 1][0][i], p, O[d], 0, 0, 0);
        if constexpr (SPLIT) {
          O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y[bi & 1][0][i], sf_bitcast<half8_t>(pl[s]), O[d], 0, 0, 0);
          O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y[bi & 1][1][i], p, O[d], 0, 0, 0);
        }
      }
    }
    if (fv & kV6) {
#pragma unroll
      for (int d = 0; d < NDB; ++d) O[d] *= fv >> 32 * d / a.g & 1 ? 64.f : 1.f;
    }
    if (fv & kVNone) {  // what is not finite, for the columns that see it
      for (int t = TS * j; t < min(TS * j + TS, lim); ++t)
#pragma unroll
        for (int d = 0; d < NDB; ++d)
          if (q4_none(a.vp[((size_t)bk * a.T_cap + t) * NG + 32 * d / a.g])) {
#pragma unroll
            for (int e = 0; e < 16; ++e) O[d][e] = NAN;
          }
    }
  };

  float16_t S0[NT], S1[NT];
  const int nit = (ntot + KG - 1) / KG;
  if (nit > 0) {
    __builtin_amdgcn_s_waitcnt((15 << 8) | (7 << 4));  // vmcnt(0)
    __syncthreads();
    load(1, false);
    score(0, 0, 2 * NFW, S0);
  }
#pragma unroll 1
  for (int it = 0; it < nit; it += 2) {
    step(it, S0, S1);
    if (it + 1 < nit) step(it + 1, S1, S0);
  }
  const float2_t lp = sf_swap32_pair(lsum);
  lsum = lp.x + lp.y;
  if constexpr (KG == 2) {
    // the odd tiles' states join the even ones' (a wave without tiles holds m = -inf, l = 0, O = 0)
    __syncthreads();  // the tiles are read
    float *const x = (float *)lds + wave * 64 * (16 * NDB + 2) + lane;
    if (kgrp) {
      x[0] = m;
      x[64] = lsum;
#pragma unroll
      for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[64 * (2 + 16 * d + e)] = O[d][e];
    }
    __syncthreads();
    if (kgrp) return;
    {
      const float m2 = x[0], M = fmaxf(m, m2), M_ref = sf_merge_mref(M);
      const float w1 = sf_merge_weight(m, M_ref), w2 = sf_merge_weight(m2, M_ref);
      lsum = fmaf(w2, x[64], w1 * lsum);
#pragma unroll
      for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) O[d][e] = fmaf(x[64 * (2 + 16 * d + e)], w2, O[d][e] * w1);
    }
  }
  if (cw + l32 >= ncol) return;
  const float inv = lsum > 0.f ? 1.f / lsum : lsum != lsum ? lsum : 0.f;
  const size_t o = qrow * D + 4 * h;
#pragma unroll
  for (int d = 0; d < NDB; ++d)
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const float4_t v = float4_t{O[d][4 * e4], O[d][4 * e4 + 1], O[d][4 * e4 + 2], O[d][4 * e4 + 3]} * inv;
      if (SPLIT && a.odt == SF_F32) {
        *(float4_t *)((float *)a.out + o + 32 * d + 8 * e4) = v;
      } else {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = SPLIT && a.odt == SF_F16 ? sf_bitcast<uint16_t>((f16)v[i]) : sf_f32_to_bf16(v[i]);
        *(u32x2 *)((uint16_t *)a.out + o + 32 * d + 8 * e4) = u32x2{u[0] | u[1] << 16, u[2] | u[3] << 16};
      }
    }
}

// The workspace of the many rows' launches where they take a call, else 0: a workgroup's walk
// takes as long whatever the number of workgroups up to one a CU, the splits' launches as
// much as the products, at any length. us, splits / many rows, of so many workgroups (of many rows):
// 32 / 8 heads of 128, one part: 2000 slots 64 38 / 44, 80 54 / 44, 128 69 / 45; 16384 slots 64 219 / 249,
// 80 312 / 250; 65536 slots 64 796 / 989, 128 1522 / 1002; no slots but the rows' own 64 13 / 17, 80 22 / 19.
// Two parts: 2000 slots 128 73 / 92, 176 95 / 96, 256 122 / 103; 16384 slots 160 559 / 618, 176 656 / 619;
// 65536 slots 128 1760 / 2490. 14 / 2 heads of 64, 16384 slots: one part 90 166 / 171, 100 208 / 171; two
// 176 341 / 385, 220 390 / 393; eight sequences in groups of 32 over 2000, two parts: 144 53 / 61, 176 65 /
// 63. Four sequences in groups of 32 over 2000, one part: 64 73 / 50. (Past 2 GiB the splits' take it.)
size_t q4_many_bytes(int B, int Tq, int H, int KVH, int T_max, int D, int parts) {
  if (D != 64 && D != 128) return 0;
  const long long blocks = (((long long)Tq * (H / KVH) + 127) / 128) * KVH * B;
  if (blocks < (parts == 1 ? 80 : 176) || (long long)Tq * (H / KVH) < 64) return 0;
  const size_t tiles = (size_t)B * KVH * q4_tiles(T_max), bytes = tiles * (2 * q4_block_bytes(D, parts) + 8);
  return bytes > (size_t)1 << 31 ? 0 : bytes;
}

// The splits of a call: none up to 12 tiles; else a tile a wave, while one sequence's workgroups go
// round the CUs once, several (ragged) sequences' as many as are resident at a time. us a call in
// a replayed graph at the rule's count (others in parentheses), 32 / 8 heads of 128, groups of 64:
// 500 slots 9.6 (1; 2: 10.7, 8: 9.9), 8191 11.1 (32; 16: 12.5, 64: 13.6), four ragged sequences up
// to 32767 32.4 (16; 8: 35.3, 12: 36.4, 24: 39.0), sixteen up to 4001 with fp32 queries 23.7 (4; 6:
// 28.3, 12: 32.0), eight up to 1000 13.1 (5; 1: 12.8, 4: 11.1, 8: 12.5); 131071 slots in groups of
// 128 31.9 (32; 16: 52.0, 96: 36.0); 14 / 2 heads of 64, 1501 slots 8.9 (6; 1: 11.3, 24: 8.7), 16384
// 9.1 (64; 16: 12.1, 128: 10.2); 40 / 2 heads of 128 in groups of 32, two up to 20000 21.8 (32; 16:
// 28.9, 48: 30.1).
int q4_splits(int B, int Tq, int H, int KVH, int T_max, int D, int group, bool split_q, int n_splits) {
  const int R = Tq * (H / KVH), PK = R <= 4 ? 4 : R <= 8 ? 2 : 1, tiles = (T_max + 63) / 64;
  const int groups = (D == 64 || D == 128) ? D / group : 0;
  const long long heads = (long long)B * KVH * (PK > 1 ? 1 : (R + 15) / 16);
  if (n_splits <= 0) {
    const long long most = (B == 1 ? 256LL : 256LL * q4_resident(D, groups, PK, split_q)) / heads;
    n_splits = tiles <= 12 ? 1 : (int)((tiles + 3) / 4 < most ? (tiles + 3) / 4 : most);
  }
  if (n_splits > tiles) n_splits = tiles;
  return n_splits > kQaMaxSplits ? kQaMaxSplits : n_splits < 1 ? 1 : n_splits;
}

// Whether P, K and V of many rows go in two parts: what an fp16 part alone loses is below a bf16
// output's rounding, but for the exponents of fp32 queries.
bool q4_whole(int q_dtype, int out_dtype) { return out_dtype != SF_BF16 || q_dtype == SF_F32; }

size_t q4_parts(long long rows, int D, int S, size_t *ml_off) {
  *ml_off = sf_align256((size_t)rows * S * D * sizeof(float));
  return S > 1 ? *ml_off + (size_t)rows * S * 2 * sizeof(float) : 0;
}

}  // namespace

extern "C" size_t sf_attn_q4_workspace_bytes(int B, int Tq, int H, int KVH, int T_max, int D, int group, int q_dtype,
                                             int out_dtype, int n_splits) {
  if (B <= 0 || Tq <= 0 || H <= 0 || KVH <= 0 || H % KVH || T_max < 0 || T_max > kQaMaxSlots || D <= 0 || group <= 0) return 0;
  size_t ml;
  if (const size_t many = q4_many_bytes(B, Tq, H, KVH, T_max, D, q4_whole(q_dtype, out_dtype) ? 2 : 1)) return many;
  return q4_parts((long long)B * Tq * H, D, q4_splits(B, Tq, H, KVH, T_max, D, group, q_dtype == SF_F32, n_splits),
                  &ml);
}

extern "C" int sf_attn_q4kv(const void *q, int q_dtype, const uint8_t *k_codes, const void *k_params,
                            const uint8_t *v_codes, const void *v_params, int group, void *out, int out_dtype,
                            void *workspace, size_t workspace_bytes, int B, int Tq, int H, int KVH,
                            const int32_t *lengths, int T, int T_max, int T_cap, int D, float scale, int n_splits,
                            void *stream) {
  SF_REQUIRE(B > 0 && Tq > 0 && H > 0 && KVH > 0 && D > 0 && T_cap > 0 && T_max >= 0 && T_max <= T_cap &&
                 (lengths || (T >= 0 && T <= T_max)),
             SF_EINVAL, "invalid attention shape B=%d Tq=%d H=%d KVH=%d T=%d T_max=%d T_cap=%d D=%d", B, Tq, H, KVH,
             T, T_max, T_cap, D);
  SF_REQUIRE(H % KVH == 0, SF_EINVAL, "n_heads=%d not a multiple of n_kv_heads=%d", H, KVH);
  if (int rc = sf_q4_cache_check(D, group)) return rc;
  SF_REQUIRE(T_max <= kQaMaxSlots, SF_EUNSUPPORTED, "T_max=%d: at most %d slots", T_max, kQaMaxSlots);
  SF_REQUIRE(isfinite(scale * 1.4426950408889634f), SF_EINVAL, "scale %g is not finite in base 2", scale);
  const long long nrb = ((long long)Tq * (H / KVH) + 15) / 16, rows = (long long)B * Tq * H;
  const size_t many = q4_many_bytes(B, Tq, H, KVH, T_max, D, q4_whole(q_dtype, out_dtype) ? 2 : 1);
  SF_REQUIRE((many ? (long long)B * KVH <= 65535 : KVH * nrb <= 65535) && B <= 65535 && rows <= 0x7fffffffLL, SF_EINVAL,
             "B=%d KVH=%d rows=%d exceed the grid", B, KVH, Tq);
  SF_REQUIRE(q_dtype >= SF_F32 && q_dtype <= SF_BF16 && out_dtype >= SF_F32 && out_dtype <= SF_BF16, SF_EINVAL,
             "bad q/out dtype");
  SF_REQUIRE(q && k_codes && k_params && v_codes && v_params && out, SF_EINVAL, "null pointer argument");
  SF_REQUIRE((((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_params | (uintptr_t)v_params | (uintptr_t)q |
               (uintptr_t)out) & 15) == 0,
             SF_EINVAL, "q, out and cache buffers must be 16-byte aligned");
  n_splits = many ? 1 : q4_splits(B, Tq, H, KVH, T_max, D, group, q_dtype == SF_F32, n_splits);
  size_t ml_off;
  const size_t parts = q4_parts(rows, D, n_splits, &ml_off), need = many ? many : parts;
  SF_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 255) == 0), SF_EINVAL, "workspace must be 256-byte aligned");
  SF_REQUIRE(workspace_bytes >= need, SF_EINVAL, "attention workspace too small: %zu < %zu", workspace_bytes, need);
  float *acc = (float *)workspace, *ml = (float *)((char *)workspace + ml_off);
  hipStream_t st = (hipStream_t)stream;
  const Q4Attn a = {q, k_codes, v_codes, (const uint32_t *)k_params, (const uint32_t *)v_params, out, acc, ml, lengths,
                    q_dtype, out_dtype, T, T_max, T_cap, Tq, H, KVH, D, group, n_splits, 0,
                    scale * 1.4426950408889634f};  // softmax in base 2
  if (many) {
    const unsigned blocks = (unsigned)((long long)B * KVH * (((long long)Tq * (H / KVH) + 127) / 128));
    const dim3 tiles((unsigned)q4_tiles(T_max), (unsigned)(B * KVH));
    uint8_t *const ws = (uint8_t *)workspace;
    Q4Attn r = a;
    r.n_splits = B * KVH;
    // The order of a head's columns where all are resident at once, one or two a CU (us, longest first /
    // the first CUs' shortest first: bf16, 32 / 8 heads of 128, 1200 rows 38.0 / 36.9, 1500 behind 300
    // 52.3 / 49.9, 2000 behind 8000 321 / 314, 40 / 2 heads 1400 behind 1000 69.5 / 64.7; fp32 1500
    // behind 300 97.6 / 95.1; 14 / 2 heads of 64, bf16, 3000 rows 49.3 / 48.8); longest first where
    // there are more.
    const int heads = B * KVH, cols = (int)(blocks / heads), per = 256 / heads;
    if (cols > per && cols <= 2 * per) r.first = per;
    // Four waves a workgroup for one part of 128 dims, where there are more workgroups than CUs: two a CU
    // between barriers of their own; else eight, which halves the longest columns' walk. us, four /
    // eight waves, bf16: 128 dims, 304 workgroups 36.9 / 35.2, 376 49.9 / 49.9, 438 64.8 / 71.5, 504 behind
    // 8000 slots 314 / 324, 1024 166 / 173, 160 65.9 / 58.3; 64 dims, 252 39.0 / 31.6, 330 49.0 / 39.4,
    // 504 72.2 / 62.0, 876 166 / 166. (Two parts at 376 110 / 104 with fp32 queries, 97 / 89 with fp16.)
    const bool four = !q4_whole(q_dtype, out_dtype) && D == 128 && blocks > 256;
#define SF_QR(QD, SP, DD)                                                                                        \
  do {                                                                                                           \
    uint32_t *const fl = (uint32_t *)(ws + tiles.x * (size_t)tiles.y * 2 * q4_block_bytes(DD, SP ? 2 : 1));      \
    k_q4_spread<SP, DD><<<tiles, 256, 0, st>>>(a, ws, fl);                                                       \
    if constexpr (!SP && DD == 128) {                                                                            \
      if (four) k_q4_rows<QD, SP, DD, 1><<<blocks, 256, 0, st>>>(r, ws, fl);                                     \
    }                                                                                                            \
    if (!four) k_q4_rows<QD, SP, DD, 2><<<blocks, 512, 0, st>>>(r, ws, fl);                                \
  } while (0)
#define SF_QR_O(QD, SP)                  \
  do {                                   \
    if (D == 64) SF_QR(QD, SP, 64);      \
    else SF_QR(QD, SP, 128);             \
  } while (0)
    if (q_dtype == SF_F32) SF_QR_O(SF_F32, true);
    else if (q_dtype == SF_F16 && out_dtype == SF_BF16) SF_QR_O(SF_F16, false);
    else if (q_dtype == SF_F16) SF_QR_O(SF_F16, true);
    else if (out_dtype == SF_BF16) SF_QR_O(SF_BF16, false);
    else SF_QR_O(SF_BF16, true);
#undef SF_QR_O
#undef SF_QR
    return sf_check_launch("sf_attn_q4kv");
  }
  const dim3 grid(n_splits, (unsigned)(KVH * nrb), B);
  const int R = Tq * (H / KVH);
#define SF_QA(QS, SG, DP, NG, KSG, PK) k_q4_split<QS, SG, DP, NG, KSG, PK><<<grid, kQaThreads, 0, st>>>(a)
#define SF_QA_R(QS, SG, DP, NG, KSG)               \
  do {                                             \
    if (R <= 4) SF_QA(QS, SG, DP, NG, KSG, 4);     \
    else if (R <= 8) SF_QA(QS, SG, DP, NG, KSG, 2); \
    else SF_QA(QS, SG, DP, NG, KSG, 1);            \
  } while (0)
#define SF_QA_D(QS, SG)                                       \
  do {                                                        \
    if (D == 64 && group == 64) SF_QA_R(QS, SG, 64, 1, 2);    \
    else if (D == 64 && group == 32) SF_QA_R(QS, SG, 64, 2, 1);    \
    else if (D == 128 && group == 128) SF_QA_R(QS, SG, 128, 1, 4); \
    else if (D == 128 && group == 64) SF_QA_R(QS, SG, 128, 2, 2);  \
    else if (D == 128 && group == 32) SF_QA_R(QS, SG, 128, 4, 1);  \
    else if (D <= 128) SF_QA(QS, SG, 128, 0, 0, 1);           \
    else SF_QA(QS, SG, 256, 0, 0, 1);                         \
  } while (0)
  if (q_dtype == SF_F32) SF_QA_D(true, true);
  else if (out_dtype != SF_BF16) SF_QA_D(false, true);
  else SF_QA_D(false, false);
#undef SF_QA_D
#undef SF_QA_R
#undef SF_QA
  if (n_splits > 1) k_q4_merge<<<(unsigned)rows, kQaThreads, 0, st>>>(acc, ml, out, out_dtype, Tq, H, KVH, D, n_splits);
  return sf_check_launch("sf_attn_q4kv");
}
