// rotary.hip — rotary positions given row by row (gfx950).
//
// A head's first r = 2 P dims are P pairs; pair i of a row at position p turns by
// the angle a = p f_i:
//   y1 = x1 c - x2 s,  y2 = x2 c + x1 s,  c = scale cos a, s = scale sin a,
// (x1, x2) = (x[i], x[i + P]) or, interleaved, (x[2 i], x[2 i + 1]). Dims past r
// stay as they are. f_i and a are held in 64 bits: at position 10^6 an fp32
// product is off by up to 0.03 of a radian. c and s are rounded to fp32, products
// and sums are fp32, the result is rounded once to the output's type.
//
//   sf_rotary            q (and k) rows, any strides, in place or not
//   sf_rotary_kv_append  q|k|v projection rows: q rotated out, k rotated and v as
//                        it is quantized (s = max|x| / 127) into int8 cache slots
//                        that need not equal the positions
#include <math.h>

#include "sf_common.h"

namespace {

// The turned pair, products and sums rounded each on its own.
__device__ __forceinline__ float2_t turn(float x1, float x2, float2_t cs) {
#pragma clang fp contract(off)
  return float2_t{x1 * cs.x - x2 * cs.y, x2 * cs.x + x1 * cs.y};
}

// cos and sin of pos * f times scale, in fp32.
__device__ __forceinline__ float2_t rotary_cs(long long pos, double f, float scale) {
  double s, c;
  sincos((double)pos * f, &s, &c);
  return float2_t{(float)(scale * c), (float)(scale * s)};
}

struct RotaryPos {
  const void *p;    // [B][T] or, stride_b = 0, [T]
  int i64;
  long long stride_b;
  __device__ __forceinline__ long long at(int b, int t) const {
    const size_t i = (size_t)b * stride_b + t;
    return i64 ? ((const long long *)p)[i] : (long long)((const int *)p)[i];
  }
};

struct RotaryRows {  // one tensor's strides in elements (batch, row, head)
  const void *in;
  void *out;
  long long ib, it, ih, ob, ot, oh;
  int heads;
};

constexpr int kRotThreads = 256;
constexpr int kRotMaxPairs = 512;

template <int DT>
__global__ void __launch_bounds__(kRotThreads)
k_rotary(RotaryRows q, RotaryRows k, RotaryPos pos, const double *__restrict__ inv_freq, int P,
         float scale, int interleaved, int T, int D) {
  __shared__ float2_t cs[kRotMaxPairs];
  const int b = blockIdx.x / T, t = blockIdx.x - b * T;
  const long long p = pos.at(b, t);
  for (int i = threadIdx.x; i < P; i += kRotThreads) cs[i] = rotary_cs(p, inv_freq[i], scale);
  __syncthreads();
  const int rest = D - 2 * P, per = P + rest;  // a head's items: pairs, then single dims
  const int n = (q.heads + k.heads) * per;
  for (int e = threadIdx.x; e < n; e += kRotThreads) {
    const int hh = e / per, i = e - hh * per;
    const RotaryRows &r = hh < q.heads ? q : k;
    const int h = hh < q.heads ? hh : hh - q.heads;
    const size_t src = (size_t)(b * r.ib + t * r.it + h * r.ih), dst = (size_t)(b * r.ob + t * r.ot + h * r.oh);
    if (i < P) {
      const int d1 = interleaved ? 2 * i : i, d2 = interleaved ? d1 + 1 : i + P;
      const float x1 = sf_load_as_f32<DT>(r.in, src + d1), x2 = sf_load_as_f32<DT>(r.in, src + d2);
      const float2_t y = turn(x1, x2, cs[i]);
      sf_store_from_f32<DT>(r.out, dst + d1, sf_opaque(y.x));
      sf_store_from_f32<DT>(r.out, dst + d2, sf_opaque(y.y));
    } else {
      const int d = P + i;
      sf_store_from_f32<DT>(r.out, dst + d, sf_load_as_f32<DT>(r.in, src + d));
    }
  }
}

struct AppendArgs {
  void *q_out;
  int8_t *k_codes, *v_codes;
  void *k_scales, *v_scales;
  int *slot_positions;  // or null
  float *scores;        // or null
  const int *lengths;   // or null: start for every sequence
  int start, q_dtype, scale_dtype, H, KVH, D, T_cap;
};

// One wave per (row, head of q|k|v). Lane l owns the pairs l and l + 64 of the head
// (D <= 256): a rotated pair, or past the rotated part two neighbouring dims.
template <int IDT>
__global__ void __launch_bounds__(64)
k_rotary_kv_append(const void *__restrict__ qkv, RotaryPos pos, const double *__restrict__ inv_freq,
                   int P, float scale, int interleaved, int T, AppendArgs a) {
  const int heads = a.H + 2 * a.KVH, head = blockIdx.x % heads, row = blockIdx.x / heads;
  const int b = row / T, t = row - b * T, lane = threadIdx.x;
  const bool is_q = head < a.H, is_v = head >= a.H + a.KVH;
  const long long p = pos.at(b, t);
  const size_t src = ((size_t)row * heads + head) * a.D;
  float x1[2], x2[2];
  int d1[2], d2[2];
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int i = lane + 64 * j;
    const bool in = 2 * i < a.D, turned = i < P;
    d1[j] = turned && !interleaved ? i : 2 * i;
    d2[j] = turned && !interleaved ? i + P : 2 * i + 1;
    x1[j] = x2[j] = 0.f;
    if (!in) continue;
    x1[j] = sf_load_as_f32<IDT>(qkv, src + d1[j]);
    x2[j] = sf_load_as_f32<IDT>(qkv, src + d2[j]);
    if (turned && !is_v) {
      const float2_t y = turn(x1[j], x2[j], rotary_cs(p, inv_freq[i], scale));
      x1[j] = y.x;
      x2[j] = y.y;
    }
    amax = fmaxf(amax, fmaxf(fabsf(x1[j]), fabsf(x2[j])));
  }
  if (is_q) {
    const size_t o = ((size_t)row * a.H + head) * a.D;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (2 * (lane + 64 * j) < a.D) {
        sf_store_dt(a.q_out, a.q_dtype, o + d1[j], sf_opaque(x1[j]));
        sf_store_dt(a.q_out, a.q_dtype, o + d2[j], sf_opaque(x2[j]));
      }
    return;
  }
  const int len = a.lengths ? a.lengths[b] : a.start;
  const long long slot = (long long)len + t;
  if (len < 0 || slot >= a.T_cap) return;  // no such slot: nothing is written
  amax = sf_wave_max(amax);
  const float s = amax == 0.f ? 1.f : amax / 127.f;
  const int kvh = is_v ? head - a.H - a.KVH : head - a.H;
  const size_t crow = ((size_t)b * a.KVH + kvh) * a.T_cap + (size_t)slot;
  int8_t *codes = (is_v ? a.v_codes : a.k_codes) + crow * a.D;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (2 * (lane + 64 * j) < a.D) {
      codes[d1[j]] = (int8_t)(int)fminf(fmaxf(__builtin_rintf(x1[j] / s), -128.f), 127.f);
      codes[d2[j]] = (int8_t)(int)fminf(fmaxf(__builtin_rintf(x2[j] / s), -128.f), 127.f);
    }
  if (lane == 0) {
    sf_store_dt(is_v ? a.v_scales : a.k_scales, a.scale_dtype, crow, s);
    if (!is_v && a.slot_positions) a.slot_positions[crow] = (int)p;
    if (!is_v && a.scores) a.scores[crow] = 0.f;
  }
}

}  // namespace

static int rotary_check(const void *positions, const double *inv_freq, int rot_pairs, int B, int T, int H,
                        int KVH, int D) {
  SF_REQUIRE(B >= 0 && T >= 0 && H > 0 && KVH >= 0 && D > 0, SF_EINVAL,
             "invalid rotary shape B=%d T=%d H=%d KVH=%d D=%d", B, T, H, KVH, D);
  SF_REQUIRE(rot_pairs > 0 && 2LL * rot_pairs <= D, SF_EINVAL, "%d rotated pairs in a head of %d", rot_pairs, D);
  SF_REQUIRE(rot_pairs <= kRotMaxPairs, SF_EUNSUPPORTED, "%d rotated pairs: at most %d", rot_pairs, kRotMaxPairs);
  SF_REQUIRE((long long)B * T == 0 || (positions && inv_freq), SF_EINVAL, "null pointer argument");
  return SF_OK;
}

extern "C" int sf_rotary(const void *q, void *q_out, const void *k, void *k_out, int dtype,
                         const void *positions, int pos_i64, int pos_per_seq, const double *inv_freq,
                         int rot_pairs, float scale, int interleaved, int B, int T, int H, int KVH, int D,
                         const long long *strides, void *stream) {
  if (int rc = rotary_check(positions, inv_freq, rot_pairs, B, T, H, KVH, D)) return rc;
  SF_REQUIRE(dtype >= SF_F32 && dtype <= SF_BF16, SF_EINVAL, "bad dtype %d", dtype);
  SF_REQUIRE((long long)B * T <= 0x7fffffffLL, SF_EINVAL, "%d x %d rows exceed the grid", B, T);
  if (B == 0 || T == 0) return SF_OK;
  SF_REQUIRE(q && q_out && (KVH == 0 || (k && k_out)), SF_EINVAL, "null pointer argument");
  const long long dq = (long long)H * D, dk = (long long)KVH * D;
  const long long whole[12] = {T * dq, dq, D, T * dq, dq, D, T * dk, dk, D, T * dk, dk, D};
  const long long *s = strides ? strides : whole;
  const RotaryRows rq = {q, q_out, s[0], s[1], s[2], s[3], s[4], s[5], H};
  const RotaryRows rk = {k, k_out, s[6], s[7], s[8], s[9], s[10], s[11], KVH};
  const RotaryPos pos = {positions, pos_i64, pos_per_seq ? T : 0};
  hipStream_t st = (hipStream_t)stream;
  const unsigned grid = (unsigned)(B * T);
#define SF_ROT(DT) k_rotary<DT><<<grid, kRotThreads, 0, st>>>(rq, rk, pos, inv_freq, rot_pairs, scale, interleaved, T, D)
  if (dtype == SF_F32) SF_ROT(SF_F32);
  else if (dtype == SF_F16) SF_ROT(SF_F16);
  else SF_ROT(SF_BF16);
#undef SF_ROT
  return sf_check_launch("sf_rotary");
}

extern "C" int sf_rotary_kv_append(const void *qkv, int in_dtype, const void *positions, int pos_i64,
                                   int pos_per_seq, const double *inv_freq, int rot_pairs, float scale,
                                   int interleaved, void *q_out, int q_dtype, int8_t *k_codes, void *k_scales,
                                   int8_t *v_codes, void *v_scales, int scale_dtype, int32_t *slot_positions,
                                   float *scores, const int32_t *lengths, int start, int B, int T, int H,
                                   int KVH, int D, int T_cap, void *stream) {
  if (int rc = rotary_check(positions, inv_freq, rot_pairs, B, T, H, KVH, D)) return rc;
  SF_REQUIRE(KVH > 0 && H % KVH == 0, SF_EINVAL, "n_heads=%d not a multiple of n_kv_heads=%d", H, KVH);
  SF_REQUIRE(D % 8 == 0 && D <= 256, SF_EUNSUPPORTED, "head_dim=%d: need D %% 8 == 0 and D <= 256", D);
  SF_REQUIRE(in_dtype >= SF_F32 && in_dtype <= SF_BF16 && q_dtype >= SF_F32 && q_dtype <= SF_BF16, SF_EINVAL,
             "bad input / q dtype");
  SF_REQUIRE(scale_dtype == SF_F16 || scale_dtype == SF_F32, SF_EINVAL, "bad scale dtype %d", scale_dtype);
  SF_REQUIRE(T_cap > 0 && (lengths || (start >= 0 && (long long)start + T <= T_cap)), SF_EINVAL,
             "KV cache overflow: %d + %d > capacity %d", start, T, T_cap);
  const long long waves = (long long)B * T * (H + 2 * KVH);
  SF_REQUIRE(waves <= 0x7fffffffLL, SF_EINVAL, "%d x %d rows exceed the grid", B, T);
  if (waves == 0) return SF_OK;
  SF_REQUIRE(qkv && q_out && k_codes && k_scales && v_codes && v_scales, SF_EINVAL, "null pointer argument");
  const RotaryPos pos = {positions, pos_i64, pos_per_seq ? T : 0};
  const AppendArgs a = {q_out, k_codes, v_codes, k_scales, v_scales, slot_positions, scores, lengths,
                        start, q_dtype, scale_dtype, H, KVH, D, T_cap};
  hipStream_t st = (hipStream_t)stream;
#define SF_ROT(DT) \
  k_rotary_kv_append<DT><<<(unsigned)waves, 64, 0, st>>>(qkv, pos, inv_freq, rot_pairs, scale, interleaved, T, a)
  if (in_dtype == SF_F32) SF_ROT(SF_F32);
  else if (in_dtype == SF_F16) SF_ROT(SF_F16);
  else SF_ROT(SF_BF16);
#undef SF_ROT
  return sf_check_launch("sf_rotary_kv_append");
}
