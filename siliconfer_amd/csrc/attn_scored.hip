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
#include <math.h>

#include "attn_common.h"
#include "sf_common.h"
#include "split_merge.h"

namespace {

constexpr int kScThreads = 256;
constexpr int kScWaves = kScThreads / 64;
constexpr int kScMaxSplits = 128;
constexpr int kScMaxRows = 32;       // query rows a sequence (Tq)
constexpr int kScTokBlock = 256;     // slots a workgroup of the weights launch

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

template <int QDT, int SDT, int DP, bool EXACT>
__global__ void __launch_bounds__(kScThreads)
k_scored_split(ScoredArgs a) {
  constexpr int KS = DP / 32, DB = DP / 16, CH = DP / 8;  // k-steps, 16-dim blocks, 8-dim chunks
  constexpr int PITCH = DP + 8;
  constexpr bool QSPLIT = QDT != SF_F16;
  constexpr int kVt = kScWaves * 32 * PITCH, kO = kScWaves * 16 * DP * 4;
  __shared__ __attribute__((aligned(16))) uint8_t smem[(kVt > kO ? kVt : kO) + 2 * kScWaves * 16 * 4];
  const int D = EXACT ? DP : a.D;
  const int G = a.H / a.KVH, R = a.Tq * G, nrb = (R + 15) / 16;
  const int split = blockIdx.x, kvh = blockIdx.y / nrb, rb = blockIdx.y - kvh * nrb, b = blockIdx.z;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane & 15, g = lane >> 4, nr = min(16, R - 16 * rb);
  const int r = 16 * rb + hl, qt = min(r, R - 1) / G, qh = min(r, R - 1) - qt * G;
  const int n = scored_len(a.lengths, a.T, a.T_max, b);
  const int lim = r < R ? max(0, n - a.Tq + qt + 1) : 0;
  const size_t bk = (size_t)b * a.KVH + kvh, base = bk * a.T_cap;

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
  auto slot_of = [&](int i) { return (i < 4 ? 4 * g + i : 16 + 4 * g + (i - 4)); };
  float4_t *sw = (float4_t *)(a.s_ws + (bk * R + 16 * rb) * (size_t)scored_tp(a.T_max));

  const int ntot = (n + 31) / 32;
  for (int j = split + a.n_splits * wave; j < ntot; j += a.n_splits * kScWaves) {
    const int tb = 32 * j;
    float4_t S[2];
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2) {
      S[h2] = float4_t{0.f, 0.f, 0.f, 0.f};
      const int8_t *kp = a.kc + (base + min(tb + 16 * h2 + hl, n - 1)) * D;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const int c = g * KS + k;
        u32x2 w = {0u, 0u};
        if (EXACT || 8 * c < D) w = *(const u32x2 *)(kp + 8 * c);
        const half8_t x = i8x8_to_h8(w.x, w.y);
        S[h2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, qh8[k], S[h2], 0, 0, 0);
        if constexpr (QSPLIT) S[h2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ql8[k], S[h2], 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < 32 * CH / 64 + (32 * CH % 64 != 0); ++i) {
      const int e = lane + 64 * i, tok = e / CH, c = e - tok * CH;
      if (tok < 32 && (EXACT || 8 * c < D))
        *(u32x2 *)(vt + tok * PITCH + 8 * c) = *(const u32x2 *)(a.vc + (base + min(tb + tok, n - 1)) * D + 8 * c);
    }
    float sc[8], vsc[8], mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = tb + slot_of(i);
      const size_t row = base + min(s, n - 1);
      vsc[i] = sf_load_as_f32<SDT>(a.vs, row);
      sc[i] = s < lim ? S[i >> 2][i & 3] * (sf_load_as_f32<SDT>(a.ks, row) * qmul) : -INFINITY;
      mx = fmaxf(mx, sc[i]);
    }
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
      // a slot past the row's weighs exactly 0 (its scale may be anything)
      pv[i] = tb + slot_of(i) < lim ? p * vsc[i] : 0.f;
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
    const int vtok = slot_of(hl >> 1);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      if (!EXACT && 16 * d >= D) break;
      typedef int v2i __attribute__((ext_vector_type(2)));
      const v2i w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
          (__attribute__((address_space(3))) v2i *)(vt + vtok * PITCH + 16 * d + 8 * (hl & 1)));
      const half8_t x = i8x8_to_h8((uint32_t)w.x, (uint32_t)w.y);
      O[d] *= oc;
      O[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ph, O[d], 0, 0, 0);
      O[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, pl, O[d], 0, 0, 0);
    }
  }
  lsum = sum_x16_x32(lsum);

  // merge the wave states through LDS into the split's partial
  __syncthreads();
  float *os = (float *)smem;  // [wave][16][DP]
  float *ms = (float *)(smem + (kVt > kO ? kVt : kO)), *ls = ms + kScWaves * 16;
  if (g == 0) {
    ms[wave * 16 + hl] = m;
    ls[wave * 16 + hl] = lsum;
  }
  const float un = 1.f / pmul;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) os[(wave * 16 + hl) * DP + 16 * d + 4 * g + i] = O[d][i] * un;
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
      acc += *(const float4_t *)(os + (w * 16 + rr) * DP + d4) * wt;
    }
    const size_t row = (bk * R + 16 * rb + rr) * a.n_splits + split;
    *(float4_t *)(a.part_acc + row * D + d4) = acc;
    if (d4 == 0) *(float2_t *)(a.part_ml + row * 2) = float2_t{M, L};
  }
}

// out = merged partials; one workgroup a query row.
__global__ void __launch_bounds__(kScThreads)
k_scored_out(const float *__restrict__ acc, const float *__restrict__ ml, void *__restrict__ out, int odt, int Tq,
             int H, int KVH, int D, int S) {
  const int G = H / KVH, R = Tq * G, row = blockIdx.x, bk = row / R, r = row - bk * R;
  const int b = bk / KVH, kvh = bk - b * KVH, t = r / G, h = r - t * G;
  const float2_t *m = (const float2_t *)ml + (size_t)row * S;
  float M = -INFINITY;
  for (int s = 0; s < S; ++s) M = fmaxf(M, m[s].x);
  const float M_ref = sf_merge_mref(M);
  const size_t o = (((size_t)b * Tq + t) * H + (size_t)kvh * G + h) * D;
  for (int d = threadIdx.x; d < D; d += kScThreads) {
    float L = 0.f, v = 0.f;
    for (int s = 0; s < S; ++s) {
      const float w = sf_merge_weight(m[s].x, M_ref);
      L = fmaf(w, m[s].y, L);
      v = fmaf(w, acc[((size_t)row * S + s) * D + d], v);
    }
    sf_store_dt(out, odt, o + d, sf_merge_finish(L, v));
  }
}

// scores += the rows' weights: a workgroup of kScTokBlock slots of one kv head.
__global__ void __launch_bounds__(kScThreads)
k_scored_weights(const float *__restrict__ s_ws, const float *__restrict__ ml, float *__restrict__ scores,
                 const int *__restrict__ lengths, int T, int T_max, int T_cap, int R, int KVH, int S) {
  extern __shared__ float sm[];  // [R] maxima, [R] reciprocal sums
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int n = scored_len(lengths, T, T_max, b), t0 = blockIdx.x * kScTokBlock;
  if (t0 >= n) return;
  const size_t bk = (size_t)b * KVH + kvh;
  for (int r = threadIdx.x; r < R; r += kScThreads) {
    const float2_t *m = (const float2_t *)ml + (bk * R + r) * S;
    float M = -INFINITY, L = 0.f;
    for (int s = 0; s < S; ++s) M = fmaxf(M, m[s].x);
    const float M_ref = sf_merge_mref(M);
    for (int s = 0; s < S; ++s) L = fmaf(sf_merge_weight(m[s].x, M_ref), m[s].y, L);
    sm[r] = M_ref;
    sm[R + r] = L > 0.f ? 1.f / L : 0.f;
  }
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hl = lane & 15, g = lane >> 4;
  const size_t tp = scored_tp(T_max);
  for (int u = wave; u < kScTokBlock / 16; u += kScWaves) {  // 16 slots: half a tile
    const int s0 = t0 + 16 * u;
    if (s0 >= n) break;
    float4_t w = {0.f, 0.f, 0.f, 0.f};
    for (int r0 = 0; r0 < R; r0 += 16) {
      const int nr = min(16, R - r0);
      if (hl >= nr) continue;
      const float4_t s = ((const float4_t *)(s_ws + (bk * R + r0) * tp))[(size_t)(s0 / 16 * 4 + g) * nr + hl];
      const float M = sm[r0 + hl], inv = sm[R + r0 + hl];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = fmaf(__builtin_amdgcn_exp2f(s[i] - M), inv, w[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // over the 16 rows: every lane gets the sum
      w[i] += sf_dpp<0xB1>(w[i]);
      w[i] += sf_dpp<0x4E>(w[i]);
      w[i] += sf_dpp<0x141>(w[i]);
      w[i] += sf_dpp<0x140>(w[i]);
    }
    const int s = s0 + 4 * g + hl;
    if (hl < 4 && s < n) {
      float *p = scores + bk * T_cap + s;
      *p += hl == 0 ? w[0] : hl == 1 ? w[1] : hl == 2 ? w[2] : w[3];
    }
  }
}

size_t scored_parts(int B, int Tq, int H, int T_max, int D, int S, size_t *ml_off, size_t *s_off) {
  const size_t rows = (size_t)B * Tq * H;
  *ml_off = sf_align256(rows * S * D * sizeof(float));
  *s_off = *ml_off + sf_align256(rows * S * 2 * sizeof(float));
  return *s_off + rows * scored_tp(T_max) * sizeof(float);
}

int scored_splits(int B, int Tq, int H, int KVH, int T_max, int D, int n_splits) {
  const int blocks = (Tq * (H / KVH) + 15) / 16;
  if (n_splits <= 0) n_splits = sf_attn_default_splits_d(B, KVH * blocks, T_max, D);
  return n_splits > kScMaxSplits ? kScMaxSplits : n_splits;
}

}  // namespace

extern "C" size_t sf_attn_scored_workspace_bytes(int B, int Tq, int H, int KVH, int T_max, int D, int n_splits) {
  if (B <= 0 || Tq <= 0 || H <= 0 || KVH <= 0 || H % KVH || T_max < 0 || D <= 0) return 0;
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
  n_splits = scored_splits(B, Tq, H, KVH, T_max, D, n_splits);
  size_t ml_off, s_off;
  const size_t need = scored_parts(B, Tq, H, T_max, D, n_splits, &ml_off, &s_off);
  SF_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0, SF_EINVAL, "workspace must be 256-byte aligned");
  SF_REQUIRE(workspace_bytes >= need, SF_EINVAL, "attention workspace too small: %zu < %zu", workspace_bytes, need);
  float *acc = (float *)workspace, *ml = (float *)((char *)workspace + ml_off), *sw = (float *)((char *)workspace + s_off);
  hipStream_t st = (hipStream_t)stream;
  const ScoredArgs a = {q, k_codes, v_codes, k_scales, v_scales, acc, ml, sw, lengths, T, T_max, T_cap, Tq, H, KVH,
                        D, n_splits, scale * 1.4426950408889634f};  // softmax in base 2
  const dim3 grid(n_splits, KVH * nrb, B);
#define SF_SC(QD, SD, DP, EX) k_scored_split<QD, SD, DP, EX><<<grid, kScThreads, 0, st>>>(a)
#define SF_SC_D(QD, SD)                         \
  do {                                          \
    if (D == 64) SF_SC(QD, SD, 64, true);       \
    else if (D == 128) SF_SC(QD, SD, 128, true); \
    else if (D <= 64) SF_SC(QD, SD, 64, false); \
    else if (D <= 128) SF_SC(QD, SD, 128, false); \
    else SF_SC(QD, SD, 256, false);             \
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
  k_scored_out<<<B * Tq * H, kScThreads, 0, st>>>(acc, ml, out, out_dtype, Tq, H, KVH, D, n_splits);
  if (T_max > 0) {
    const dim3 wgrid((T_max + kScTokBlock - 1) / kScTokBlock, KVH, B);
    k_scored_weights<<<wgrid, kScThreads, 2 * R * sizeof(float), st>>>(sw, ml, scores, lengths, T, T_max, T_cap, R,
                                                                      KVH, n_splits);
  }
  return sf_check_launch("sf_attn_decode_scored_i8kv");
}
