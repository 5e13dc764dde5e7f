// attn_scored.hip — decode attention that scores its cache (gfx950).
//
// For Tq query rows a sequence (row t sees the first n - Tq + t + 1 of its n slots)
// over an int8 cache with a scale a token and kv head:
//   w = softmax(scale q K^T),  out = w V,
//   scores[b, kvh, slot] += sum of w[slot] over the Tq rows and the kv head's
//                           query heads (R = Tq H / KVH query rows),
// the accumulated attention weight by which a bounded cache chooses what it keeps.
//
// A weight needs its row's maximum and sum over every slot, which no split of the
// slots has before all of them are done. The split launch therefore leaves, beside
// its partials (m, l, acc), the fp32 scores themselves: 4 R bytes a slot and kv head
// beside the 2 D code bytes that were read for them, still in the cache when the
// second launch turns them into weights and sums them over the rows.
//
// k_scored_split: one workgroup a (split, kv head and 16 of its rows, sequence); its
// four waves take 32-slot tiles. S^T = K q^T and O^T = V^T P^T on
// v_mfma_f32_16x16x32_f16 with the query rows on the 16-wide side, the codes exact in
// fp16, q and P as fp16 high and low parts (fp16 q is exact as it is):
//   * q of other types is first brought to a largest magnitude of 2^13..2^14 by a
//     power of two a row, P times the V scale likewise by the largest one that the
//     row has met, so neither leaves fp16's range and what the low part drops is below
//     2^-22 of the value and 2^-38 of the row's largest;
//   * lane l holds row l % 16 and slots 4 g + i, 16 + 4 g + i of a tile (g = l / 16),
//     the C layout of S^T; the same eight slots are its B operand of O^T, V^T comes
//     through LDS with ds_read_b64_tr_b8.
// Measured (us, split + finishing launch): 1501 slots at 14/2 heads of 64 4.2 + 3.8; four
// ragged sequences of up to 8191 (50 MB of cache, 10.2 us at a copy's rate) at 32/8 heads
// of 128 16.3 + 5.5, from 24.8 + 15.3 with loads and math of a tile in turn, two merge
// launches and a serial loop over the splits. VALU issue is 44% of the split's time (the
// conversion of codes and the softmax of 16 rows where a kv head has 4), the rest launch,
// first loads and the merge of its waves.
#include <math.h>

#include "attn_common.h"
#include "sf_common.h"
#include "split_merge.h"

namespace {

constexpr int kScThreads = 256;
constexpr int kScWaves = kScThreads / 64;
constexpr int kScMaxSplits = 128;
constexpr int kScMaxRows = 32;       // query rows a sequence (Tq)
constexpr int kScMaxSlots = 0x7fffff00;  // a slot number rounded up to a block of 256 stays an int

struct ScoredArgs {
  const void *q;
  const int8_t *kc, *vc;
  const void *ks, *vs;
  float *part_acc, *part_ml, *s_ws;
  const int *lengths;
  int T, T_max, T_cap, Tq, H, KVH, D, n_splits;
  float qscale;
};

__device__ __forceinline__ int scored_len(const int *lengths, int T, int T_max, int b) {
  const long long n = (long long)(lengths ? lengths[b] : 0) + T;
  return n < 0 ? 0 : n > T_max ? T_max : (int)n;
}
__host__ __device__ inline int scored_tp(int T_max) { return (T_max + 31) & ~31; }

// The power of two that takes a magnitude v to [2^13, 2^14) (1 for 0, and within the
// range of fp32's exponents).
__device__ __forceinline__ float fit14(float v) {
  const int e = (int)(sf_bitcast<uint32_t>(v) >> 23 & 255);  // 2^(e - 127) <= v
  const int f = 127 + 13 + 127 - e;
  return v == 0.f ? 1.f : sf_bitcast<float>((uint32_t)(f < 1 ? 1 : f > 253 ? 253 : f) << 23);
}

// N words at a scale's alignment: rows of a cache of any capacity start there.
template <int N>
struct __attribute__((packed, aligned(2))) Words {
  uint32_t w[N];
};

template <int QDT, int SDT, int DP, bool EXACT>
__global__ void __launch_bounds__(kScThreads, DP > 128 ? 1 : 3)
k_scored_split(ScoredArgs a) {
  constexpr int KS = DP / 32, DB = DP / 16, CH = DP / 8;  // k-steps, 16-dim blocks, 8-dim chunks
  constexpr int VC = EXACT ? DP / 32 : DP / 16;           // a lane's 16- (8-) byte pieces of a V tile
  constexpr int PITCH = DP + 8;
  constexpr bool QSPLIT = QDT != SF_F16;
  constexpr int OP = DP + 4;                              // a row's floats in LDS: 16-byte writes without conflicts
  constexpr int kVt = kScWaves * 32 * PITCH, kO = kScWaves * 16 * OP * 4;
  __shared__ __attribute__((aligned(16))) uint8_t smem[(kVt > kO ? kVt : kO) + 2 * kScWaves * 16 * 4];
  const int D = EXACT ? DP : a.D;
  const int G = a.H / a.KVH, R = a.Tq * G, nrb = (R + 15) / 16;
  const int split = blockIdx.x, kvh = blockIdx.y / nrb, rb = blockIdx.y - kvh * nrb, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane & 15, g = lane >> 4, nr = min(16, R - 16 * rb);
  const int r = 16 * rb + hl, qt = min(r, R - 1) / G, qh = min(r, R - 1) - qt * G;
  const size_t bk = (size_t)b * a.KVH + kvh, base = bk * a.T_cap;
  auto slot_of = [&](int i) { return (i < 4 ? 4 * g + i : 16 + 4 * g + (i - 4)); };

  struct Tile {
    u32x2 k[2][KS];  // the K codes of slots hl and 16 + hl, dims 8 (KS g + k) .. + 7
    u32x4 v[VC];     // V codes for the LDS stage (8 bytes of each used where !EXACT)
    u32x4 kw[2], vw[2];  // scale bits of the lane's slots 4 h2 .. + 3: four words, or two fp16 pairs
  };
  // Rows are clamped into the cache; what lies past the length is masked.
  Tile t;
  auto load_k = [&](int j) {
    const int tb = 32 * j;
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2) {
      const int8_t *kp = a.kc + (base + min(tb + 16 * h2 + hl, a.T_cap - 1)) * D;
      if constexpr (EXACT) {
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          const u32x4 w = *(const u32x4 *)(kp + 8 * (g * KS + k));
          t.k[h2][k] = u32x2{w.x, w.y};
          t.k[h2][k + 1] = u32x2{w.z, w.w};
        }
      } else {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const int c = g * KS + k;
          t.k[h2][k] = 8 * c < D ? *(const u32x2 *)(kp + 8 * c) : u32x2{0u, 0u};
        }
      }
    }
  };
  auto load_v = [&](int j) {
    const int tb = 32 * j;
#pragma unroll
    for (int i = 0; i < VC; ++i) {
      const int e = lane + 64 * i;
      if constexpr (EXACT) {
        const int tok = e / (DP / 16), c = e % (DP / 16);
        t.v[i] = *(const u32x4 *)(a.vc + (base + min(tb + tok, a.T_cap - 1)) * D + 16 * c);
      } else {
        const int tok = e / CH, c = e % CH;
        if (8 * c < D) {
          const u32x2 w = *(const u32x2 *)(a.vc + (base + min(tb + tok, a.T_cap - 1)) * D + 8 * c);
          t.v[i].x = w.x;
          t.v[i].y = w.y;
        }
      }
    }
  };
  auto load_scales = [&](int j) {
    const int tb = 32 * j;
    if (tb + 32 <= a.T_cap) {  // four slots' scales a load
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {
        const size_t row = base + tb + 16 * h2 + 4 * g;
        if constexpr (SDT == SF_F16) {
          const Words<2> x = *(const Words<2> *)((const f16 *)a.ks + row), y = *(const Words<2> *)((const f16 *)a.vs + row);
          t.kw[h2] = u32x4{x.w[0], x.w[1], 0u, 0u};
          t.vw[h2] = u32x4{y.w[0], y.w[1], 0u, 0u};
        } else {
          const Words<4> x = *(const Words<4> *)((const float *)a.ks + row), y = *(const Words<4> *)((const float *)a.vs + row);
          t.kw[h2] = u32x4{x.w[0], x.w[1], x.w[2], x.w[3]};
          t.vw[h2] = u32x4{y.w[0], y.w[1], y.w[2], y.w[3]};
        }
      }
    } else {  // the cache's last slots
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const size_t row = base + min(tb + 16 * h2 + 4 * g + i, a.T_cap - 1);
          if constexpr (SDT == SF_F16) {
            const uint32_t x = ((const uint16_t *)a.ks)[row], y = ((const uint16_t *)a.vs)[row];
            t.kw[h2][i >> 1] = i & 1 ? t.kw[h2][i >> 1] | x << 16 : x;
            t.vw[h2][i >> 1] = i & 1 ? t.vw[h2][i >> 1] | y << 16 : y;
          } else {
            t.kw[h2][i] = ((const uint32_t *)a.ks)[row];
            t.vw[h2][i] = ((const uint32_t *)a.vs)[row];
          }
        }
    }
  };
  auto scale_of = [&](const u32x4 (&w)[2], int i) {
    if constexpr (SDT == SF_F32) return sf_bitcast<float>(w[i >> 2][i & 3]);
    else return (float)sf_bitcast<f16>((uint16_t)(w[i >> 2][(i >> 1) & 1] >> (16 * (i & 1))));
  };

  const int n = scored_len(a.lengths, a.T, a.T_max, b), ntot = (n + 31) / 32;
  const int j0 = split + a.n_splits * wave, jstep = a.n_splits * kScWaves;
  if (j0 < ntot) {
    load_k(j0);
    load_scales(j0);
    load_v(j0);
  }
  const int lim = r < R ? max(0, n - a.Tq + qt + 1) : 0, lim_all = n - a.Tq + 16 * rb / G + 1;  // (of every row)
  half8_t qh8[KS], ql8[KS];
  float qmul = a.qscale;
  {
    float f[KS][8], top = 0.f;
    const size_t q0 = (((size_t)b * a.Tq + qt) * a.H + (size_t)kvh * G + qh) * D;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int c = g * KS + k;
      if (EXACT || 8 * c < D) sf_load8_as_f32<QDT>(a.q, q0 + 8 * c, f[k]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[k][i] = r < R && (EXACT || 8 * c < D) ? f[k][i] : 0.f;
        top = fmaxf(top, fabsf(f[k][i]));
      }
    }
    float up = 1.f;
    if constexpr (QSPLIT) {
      up = fit14(max_x16_x32(top));
      qmul = a.qscale / up;
    }
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = f[k][i] * up;
        qh8[k][i] = (f16)v;
        ql8[k][i] = (f16)(v - (float)qh8[k][i]);
      }
  }

  uint8_t *vt = smem + wave * 32 * PITCH;
  float m = -INFINITY, lsum = 0.f;  // base-2 softmax of row r
  float pmax = 0.f, pmul = 1.f;     // largest weight times V scale so far (as the weights stand), its factor
  float4_t O[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) O[d] = float4_t{0.f, 0.f, 0.f, 0.f};
  float4_t *sw = (float4_t *)(a.s_ws + (bk * R + 16 * rb) * (size_t)scored_tp(a.T_max));

  // A tile's registers are loaded again as soon as their bytes are in operands or in LDS:
  // the next tile flies during this one's softmax and products, at the registers and the
  // code of one tile (two tiles' code costs more in instruction fetches than it hides).
  for (int j = j0; j < ntot; j += jstep) {
    const int tb = 32 * j;
    const bool more = j + jstep < ntot;
    float4_t S[2];
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2) {
      S[h2] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const half8_t x = i8x8_to_h8(t.k[h2][k].x, t.k[h2][k].y);
        S[h2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, qh8[k], S[h2], 0, 0, 0);
        if constexpr (QSPLIT) S[h2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ql8[k], S[h2], 0, 0, 0);
      }
    }
    if (more) load_k(j + jstep);
    float sc[8], vsc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sc[i] = scale_of(t.kw, i) * qmul;
      vsc[i] = scale_of(t.vw, i);
    }
    if (more) load_scales(j + jstep);
#pragma unroll
    for (int i = 0; i < VC; ++i) {
      const int e = lane + 64 * i;
      if constexpr (EXACT) {
        uint2 *dst = (uint2 *)(vt + (e / (DP / 16)) * PITCH + 16 * (e % (DP / 16)));
        dst[0] = uint2{t.v[i].x, t.v[i].y};
        dst[1] = uint2{t.v[i].z, t.v[i].w};
      } else {
        if (8 * (e % CH) < D) *(uint2 *)(vt + (e / CH) * PITCH + 8 * (e % CH)) = uint2{t.v[i].x, t.v[i].y};
      }
    }
    if (more) load_v(j + jstep);
#pragma unroll
    for (int i = 0; i < 8; ++i) sc[i] *= S[i >> 2][i & 3];
    if (tb + 32 > lim_all) {  // a row ends here: what lies past it weighs exactly 0, whatever its scales hold
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = tb + slot_of(i) < lim;
        sc[i] = in ? sc[i] : -INFINITY;
        vsc[i] = in ? vsc[i] : 0.f;
      }
    }
    float mx = sc[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, sc[i]);
    if (hl < nr) {
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2)
        sw[(size_t)((j * 2 + h2) * 4 + g) * nr + hl] = float4_t{sc[4 * h2], sc[4 * h2 + 1], sc[4 * h2 + 2], sc[4 * h2 + 3]};
    }
    const float m_new = fmaxf(m, max_x16_x32(mx)), m_ref = m_new == -INFINITY ? 0.f : m_new;
    const float c = __builtin_amdgcn_exp2f(m - m_ref);
    m = m_new;
    float pv[8], ps = 0.f, pt = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float p = __builtin_amdgcn_exp2f(sc[i] - m_ref);
      ps += p;
      pv[i] = p * vsc[i];
      pt = fmaxf(pt, fabsf(pv[i]));
    }
    lsum = fmaf(lsum, c, ps);
    pmax = fmaxf(pmax * c, max_x16_x32(pt));
    const float mul = fit14(pmax), oc = c * mul / pmul;  // at most 2: pmax covers c times the last one
    pmul = mul;
    half8_t ph, pl;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = sf_opaque(pv[i] * mul);
      ph[i] = (f16)v;
      pl[i] = (f16)(v - (float)ph[i]);
    }
    if (__any(oc != 1.f)) {  // few tiles move a maximum
#pragma unroll
      for (int d = 0; d < DB; ++d) O[d] *= oc;
    }
    const int vtok = slot_of(hl >> 1);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      if (!EXACT && 16 * d >= D) break;
      typedef int v2i __attribute__((ext_vector_type(2)));
      const v2i w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
          (__attribute__((address_space(3))) v2i *)(vt + vtok * PITCH + 16 * d + 8 * (hl & 1)));
      const half8_t x = i8x8_to_h8((uint32_t)w.x, (uint32_t)w.y);
      O[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ph, O[d], 0, 0, 0);
      O[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, pl, O[d], 0, 0, 0);
    }
  }
  lsum = sum_x16_x32(lsum);

  // merge the wave states through LDS into the split's partial
  __syncthreads();
  float *os = (float *)smem;  // [wave][16][OP]
  float *ms = (float *)(smem + (kVt > kO ? kVt : kO)), *ls = ms + kScWaves * 16;
  if (g == 0) {
    ms[wave * 16 + hl] = m;
    ls[wave * 16 + hl] = lsum;
  }
  const float un = 1.f / pmul;
#pragma unroll
  for (int d = 0; d < DB; ++d) *(float4_t *)(os + (wave * 16 + hl) * OP + 16 * d + 4 * g) = O[d] * un;
  __syncthreads();
  const int nq = D / 4;
  for (int e = tid; e < nr * nq; e += kScThreads) {
    const int rr = e / nq, d4 = (e - rr * nq) * 4;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kScWaves; ++w) M = fmaxf(M, ms[w * 16 + rr]);
    const float M_ref = sf_merge_mref(M);
    float L = 0.f;
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kScWaves; ++w) {
      const float wt = sf_merge_weight(ms[w * 16 + rr], M_ref);
      L = fmaf(wt, ls[w * 16 + rr], L);
      acc += *(const float4_t *)(os + (w * 16 + rr) * OP + d4) * wt;
    }
    const size_t row = (bk * R + 16 * rb + rr) * a.n_splits + split;
    *(float4_t *)(a.part_acc + row * D + d4) = acc;
    if (d4 == 0) *(float2_t *)(a.part_ml + row * 2) = float2_t{M, L};
  }
}

// The second launch. Its first workgroups merge a query row's partials each: every thread
// four dims of some of the splits, the parts then summed in LDS, all loads of a thread in
// flight at once. The others turn the scores of 64 U slots of one kv head into
// weights: 16 lanes a row find its maximum and sum over the splits, then a wave takes 16
// slots at a time, lane l the four slots 4 (l / 16) .. of row l % 16, and sums the rows
// across its lanes. No atomics: the order is fixed.
struct FinishArgs {
  const float *acc, *ml, *s_ws;
  float *scores;
  void *out;
  const int *lengths;
  int odt, T, T_max, T_cap, Tq, H, KVH, D, S, tok_blocks;
};

__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, sf_dpp<0xB1>(v));
  v = fmaxf(v, sf_dpp<0x4E>(v));
  v = fmaxf(v, sf_dpp<0x141>(v));
  return fmaxf(v, sf_dpp<0x140>(v));
}
__device__ __forceinline__ float row16_sum(float v) {
  v += sf_dpp<0xB1>(v);
  v += sf_dpp<0x4E>(v);
  v += sf_dpp<0x141>(v);
  return v + sf_dpp<0x140>(v);
}

__device__ void scored_out(const FinishArgs &a, int row, float *sm) {
  constexpr int kPre = 4;  // a thread's splits loaded ahead
  const int S = a.S, nq = a.D / 4, parts = kScThreads / nq, q = threadIdx.x % nq, part = threadIdx.x / nq;
  const int lane = threadIdx.x & 63;
  const float2_t *ml = (const float2_t *)a.ml + (size_t)row * S;
  const float4_t *acc = (const float4_t *)a.acc + (size_t)row * S * nq + q;
  const float2_t e0 = ml[min(lane, S - 1)], e1 = ml[min(lane + 64, S - 1)];  // (S <= 128; every wave alike)
  float4_t pre[kPre];
#pragma unroll
  for (int k = 0; k < kPre; ++k) pre[k] = acc[(size_t)min(part + k * parts, S - 1) * nq];
  const float m0 = lane < S ? e0.x : -INFINITY, m1 = lane + 64 < S ? e1.x : -INFINITY;
  const float M = sf_merge_mref(sf_wave_max(fmaxf(m0, m1)));
  const float w0 = sf_merge_weight(m0, M), w1 = sf_merge_weight(m1, M);
  const float L = sf_wave_sum((lane < S ? w0 * e0.y : 0.f) + (lane + 64 < S ? w1 * e1.y : 0.f));
  float *w = sm;                                   // [128]
  float4_t *p = (float4_t *)(sm + kScMaxSplits);   // [parts][nq]
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
    const int G = a.H / a.KVH, R = a.Tq * G, bk = row / R, r = row - bk * R;
    const int b = bk / a.KVH, t = r / G, h = (bk - b * a.KVH) * G + r - t * G;
    const size_t o = (((size_t)b * a.Tq + t) * a.H + h) * a.D + 4 * q;
#pragma unroll
    for (int i = 0; i < 4; ++i) sf_store_dt(a.out, a.odt, o + i, sf_merge_finish(L, v[i]));
  }
}

// U units of 16 slots a wave.
template <int U>
__device__ void scored_weights(const FinishArgs &a, int blk, float *sm) {
  const int R = a.Tq * (a.H / a.KVH), S = a.S;
  const int bk = blk / a.tok_blocks, t0 = (blk - bk * a.tok_blocks) * (16 * kScWaves * U), b = bk / a.KVH;
  const int n = scored_len(a.lengths, a.T, a.T_max, b);
  if (t0 >= n) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hl = lane & 15, g = lane >> 4;
  const size_t tp = scored_tp(a.T_max);
  const float4_t *sw = (const float4_t *)(a.s_ws + (size_t)bk * R * tp);
  float *sc = a.scores + (size_t)bk * a.T_cap;
  // the unit's scores of 16 rows: (lanes past the rows read the last one's and drop it)
  auto load = [&](int s0, int r0) {
    const int nr = min(16, R - r0);
    return sw[r0 * (tp / 4) + (size_t)(s0 / 16 * 4 + g) * nr + min(hl, nr - 1)];
  };
  float4_t s[U];
  float old[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int s0 = t0 + 16 * (wave + kScWaves * u);
    s[u] = load(min(s0, n - 1) & ~15, 0);
    old[u] = sc[min(s0 + 4 * g + (hl & 3), n - 1)];
  }
  const float2_t *ml = (const float2_t *)a.ml + (size_t)bk * R * S;
  for (int r = threadIdx.x >> 4; r < ((R + 15) & ~15); r += kScThreads / 16) {
    const float2_t *e = ml + (size_t)min(r, R - 1) * S;
    constexpr int NV = kScMaxSplits / 16;
    float2_t v[NV];
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (16 * i < S) v[i] = e[min(hl + 16 * i, S - 1)];
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (16 * i < S && hl + 16 * i < S) M = fmaxf(M, v[i].x);
    M = sf_merge_mref(row16_max(M));
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (16 * i < S && hl + 16 * i < S) L += sf_merge_weight(v[i].x, M) * v[i].y;
    L = row16_sum(L);
    if (hl == 0 && r < R) {
      sm[2 * r] = M;
      sm[2 * r + 1] = L > 0.f ? 1.f / L : 0.f;
    }
  }
  __syncthreads();
  float4_t w[U];
#pragma unroll
  for (int u = 0; u < U; ++u) w[u] = float4_t{0.f, 0.f, 0.f, 0.f};
  for (int r0 = 0; r0 < R; r0 += 16) {
    const bool in = hl < R - r0;
    const float2_t mi = ((const float2_t *)sm)[min(r0 + hl, R - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s0 = t0 + 16 * (wave + kScWaves * u);
      const float4_t x = s[u];
      if (r0 + 16 < R) s[u] = load(min(s0, n - 1) & ~15, r0 + 16);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (in) w[u][i] = fmaf(__builtin_amdgcn_exp2f(x[i] - mi.x), mi.y, w[u][i]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[u][i] = row16_sum(w[u][i]);
    const int at = t0 + 16 * (wave + kScWaves * u) + 4 * g + hl;
    if (hl < 4 && at < n) sc[at] = old[u] + (hl == 0 ? w[u][0] : hl == 1 ? w[u][1] : hl == 2 ? w[u][2] : w[u][3]);
  }
}

template <int U>
__global__ void __launch_bounds__(kScThreads)
k_scored_finish(FinishArgs a, int rows) {
  extern __shared__ __attribute__((aligned(16))) float sm[];
  if ((int)blockIdx.x < rows) scored_out(a, blockIdx.x, sm);
  else scored_weights<U>(a, blockIdx.x - rows, sm);
}

size_t scored_parts(int B, int Tq, int H, int T_max, int D, int S, size_t *ml_off, size_t *s_off) {
  const size_t rows = (size_t)B * Tq * H;
  *ml_off = sf_align256(rows * S * D * sizeof(float));
  *s_off = *ml_off + sf_align256(rows * S * 2 * sizeof(float));
  return *s_off + rows * scored_tp(T_max) * sizeof(float);
}

// The decode attention's rule, with a block of 16 query rows a kv head. Measured for these kernels
// (us a call in a replayed graph, both launches, at the rule's count; other counts in
// parentheses), 14 / 2 heads of 64, fp16: 500 slots 7.1 (16; 4: 7.3, 8: 7.1); 1501 7.2 (47; 12: 7.3, 32:
// 7.1); 4096 7.2 (64; 32: 7.4, 96: 8.0); 16384 9.9 (128; 48: 9.9, 64: 9.2); 16 fp32 rows over 2000
// 15.8 (19; 8: 14.8, 16: 14.1, 32: 15.4). 32 / 8 heads of 128, bf16: 2000 9.3 (32; 16: 9.4, 48: 11.4);
// 8191 14.9 (64; 32: 14.1, 128: 19.5); four ragged sequences of 1000 10.0 (8; 4: 11.4, 16: 11.2), of
// 8191 23.5 (16; 8: 27.7, 24: 23.2, 32: 24.4); eight of 2001, fp32, 16.3 (8; 4: 17.8, 16: 18.2); sixteen of 4000
// 35.4 (4; 2: 42.3, 6: 35.1, 8: 35.7). 32 / 32 heads, four of 2000 21.7 (4; 2: 26.1, 8: 23.4).
int scored_splits(int B, int Tq, int H, int KVH, int T_max, int D, int n_splits) {
  const int blocks = (Tq * (H / KVH) + 15) / 16;
  if (n_splits <= 0) n_splits = sf_attn_default_splits_d(B, KVH * blocks, T_max, D);
  return n_splits > kScMaxSplits ? kScMaxSplits : n_splits;
}

}  // namespace

extern "C" size_t sf_attn_scored_workspace_bytes(int B, int Tq, int H, int KVH, int T_max, int D, int n_splits) {
  if (B <= 0 || Tq <= 0 || H <= 0 || KVH <= 0 || H % KVH || T_max < 0 || T_max > kScMaxSlots || D <= 0) return 0;
  size_t ml, s;
  return scored_parts(B, Tq, H, T_max, D, scored_splits(B, Tq, H, KVH, T_max, D, n_splits), &ml, &s);
}

extern "C" int sf_attn_decode_scored_i8kv(const void *q, int q_dtype, const int8_t *k_codes, const void *k_scales,
                                          const int8_t *v_codes, const void *v_scales, int scale_dtype,
                                          float *scores, void *out, int out_dtype, void *workspace,
                                          size_t workspace_bytes, int B, int Tq, int H, int KVH,
                                          const int32_t *lengths, int T, int T_max, int T_cap, int D, float scale,
                                          int n_splits, void *stream) {
  SF_REQUIRE(B > 0 && Tq > 0 && H > 0 && KVH > 0 && D > 0 && T_cap > 0 && T_max >= 0 && T_max <= T_cap &&
                 (lengths || (T >= 0 && T <= T_max)),
             SF_EINVAL, "invalid attention shape B=%d Tq=%d H=%d KVH=%d T=%d T_max=%d T_cap=%d D=%d", B, Tq, H, KVH,
             T, T_max, T_cap, D);
  SF_REQUIRE(H % KVH == 0, SF_EINVAL, "n_heads=%d not a multiple of n_kv_heads=%d", H, KVH);
  SF_REQUIRE(D <= 256, SF_EINVAL, "head_dim=%d exceeds kernel's compile-time max 256", D);
  SF_REQUIRE(D % 8 == 0, SF_EUNSUPPORTED, "head_dim=%d: need a multiple of 8", D);
  SF_REQUIRE(Tq <= kScMaxRows, SF_EUNSUPPORTED, "%d query rows a sequence: at most %d", Tq, kScMaxRows);
  SF_REQUIRE(T_max <= kScMaxSlots, SF_EUNSUPPORTED, "T_max=%d: at most %d slots", T_max, kScMaxSlots);
  const int G = H / KVH;
  SF_REQUIRE(G <= 128, SF_EUNSUPPORTED, "%d query heads a kv head: at most 128", G);
  const int R = Tq * G, nrb = (R + 15) / 16;
  SF_REQUIRE((long long)KVH * nrb <= 65535 && B <= 65535 && (long long)B * Tq * H <= 0x7fffffffLL, SF_EINVAL,
             "B=%d KVH=%d rows=%d exceed the grid", B, KVH, R);
  SF_REQUIRE(q_dtype >= SF_F32 && q_dtype <= SF_BF16 && out_dtype >= SF_F32 && out_dtype <= SF_BF16, SF_EINVAL,
             "bad q/out dtype");
  SF_REQUIRE(scale_dtype == SF_F16 || scale_dtype == SF_F32, SF_EINVAL, "bad scale dtype %d", scale_dtype);
  SF_REQUIRE(q && k_codes && k_scales && v_codes && v_scales && scores && out, SF_EINVAL, "null pointer argument");
  SF_REQUIRE((((uintptr_t)k_codes | (uintptr_t)v_codes) & 7) == 0, SF_EINVAL,
             "KV code buffers must be 8-byte aligned");
  SF_REQUIRE(((uintptr_t)q & 15) == 0, SF_EINVAL, "q must be 16-byte aligned");
  // 256 slots a workgroup of the second launch where that gives every CU two, else 64. us a call
  // with 256 / 64, shapes as above: 128 workgroups of 256 (one sequence of 16384, 2 kv heads) 9.7 / 9.9,
  // 12 of them 7.7 / 7.3, 16 rows 18.9 / 15.8; 256 (8191, 8 kv heads) 14.7 / 15.1; 512 16.7 / 18.2;
  // 1024 23.9 / 26.6 and 22.3 / 25.1.
  const bool many = (long long)B * KVH * ((T_max + 255) / 256) >= 512;
  const int rows = B * Tq * H, per = many ? 256 : 64, tok_blocks = (T_max + per - 1) / per;
  SF_REQUIRE((long long)B * KVH * tok_blocks + rows <= 0x7fffffffLL, SF_EINVAL, "B=%d T_max=%d exceed the grid", B, T_max);
  n_splits = scored_splits(B, Tq, H, KVH, T_max, D, n_splits);
  size_t ml_off, s_off;
  const size_t need = scored_parts(B, Tq, H, T_max, D, n_splits, &ml_off, &s_off);
  SF_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0, SF_EINVAL, "workspace must be 256-byte aligned");
  SF_REQUIRE(workspace_bytes >= need, SF_EINVAL, "attention workspace too small: %zu < %zu", workspace_bytes, need);
  float *acc = (float *)workspace, *ml = (float *)((char *)workspace + ml_off), *sw = (float *)((char *)workspace + s_off);
  hipStream_t st = (hipStream_t)stream;
  // codes in 16-byte pieces at D = 64 / 128
  const bool wide = (((uintptr_t)k_codes | (uintptr_t)v_codes) & 15) == 0;
  const ScoredArgs a = {q, k_codes, v_codes, k_scales, v_scales, acc, ml, sw, lengths, T, T_max, T_cap, Tq, H, KVH,
                        D, n_splits, scale * 1.4426950408889634f};  // softmax in base 2
  const dim3 grid(n_splits, KVH * nrb, B);
#define SF_SC(QD, SD, DP, EX) k_scored_split<QD, SD, DP, EX><<<grid, kScThreads, 0, st>>>(a)
#define SF_SC_D(QD, SD)                               \
  do {                                                \
    if (D == 64 && wide) SF_SC(QD, SD, 64, true);     \
    else if (D == 128 && wide) SF_SC(QD, SD, 128, true); \
    else if (D <= 64) SF_SC(QD, SD, 64, false);       \
    else if (D <= 128) SF_SC(QD, SD, 128, false);     \
    else SF_SC(QD, SD, 256, false);                   \
  } while (0)
#define SF_SC_S(QD)                                 \
  do {                                              \
    if (scale_dtype == SF_F16) SF_SC_D(QD, SF_F16); \
    else SF_SC_D(QD, SF_F32);                       \
  } while (0)
  if (q_dtype == SF_F32) SF_SC_S(SF_F32);
  else if (q_dtype == SF_F16) SF_SC_S(SF_F16);
  else SF_SC_S(SF_BF16);
#undef SF_SC_S
#undef SF_SC_D
#undef SF_SC
  const FinishArgs f = {acc, ml, sw, scores, out, lengths, out_dtype, T, T_max, T_cap, Tq, H, KVH, D, n_splits, tok_blocks};
  // LDS: the splits' weights and the parts' sums, or two words a row
  const size_t lds_out = (kScMaxSplits + 4 * kScThreads) * sizeof(float), lds_w = 2 * (size_t)R * sizeof(float);
  const size_t lds = lds_out > lds_w ? lds_out : lds_w;
  if (many) k_scored_finish<4><<<rows + B * KVH * tok_blocks, kScThreads, lds, st>>>(f, rows);
  else k_scored_finish<1><<<rows + B * KVH * tok_blocks, kScThreads, lds, st>>>(f, rows);
  return sf_check_launch("sf_attn_decode_scored_i8kv");
}
