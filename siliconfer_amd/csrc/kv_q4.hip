// kv_q4.hip — a KV cache held in 4 bits: append and reading back (gfx950).
//
// A head's D dims of a token are cut into groups of g; a group holds
//   m = f16(min x),  s = f16((max x - min x) / 15),
//   code = clip(rint((x - m) / s), 0, 15)  (0 where s is 0),  x ~ m + s code,
// codes two a byte (the even dim in the low half), (s, m) one 32-bit word a group. Beside
// the int8 cache's D + 2 bytes a head and token this is D / 2 + 4 D / g.
//
//   sf_kv_q4_append   q|k|v rows: q and k (normed a head and) turned as in qk_norm.hip, q out,
//                     k and v into slots that need not be the positions
//   sf_kv_q4_dequant  codes back to values
//
// Everything up to the code is held in 64 bits, where a wave's operation takes as long
// as an unpacked 32-bit one: a value next to a code's border then takes the same code
// whatever order the sums and products took, and the rounding of the division is settled by
// its remainder, exact in 64 bits. L lanes hold a head, 8 dims each.
#include <math.h>

#include "rotary_common.h"

namespace {

constexpr int kQ4Threads = 256;
constexpr int kQ4MaxD = 256;

struct Q4Rows {
  const void *x;          // [B, T, heads, D] by strides (elements), or null
  long long sb, st, sh;
};

struct Q4Append {
  Q4Rows q, k, v;
  const void *qw, *kw;    // norm weights, or null
  void *q_out;
  uint8_t *kc, *vc;
  uint32_t *kp, *vp;      // (s, m)
  const int *lengths;     // or null: start for every sequence
  int start, q_dtype, w_dtype, H, KVH, D, g, T, T_cap, P, interleaved, lanes_log2, n_heads;
  float eps, scale;
};

__device__ __forceinline__ double q4_load(const void *p, int dt, size_t i) {
  return dt == SF_F32 ? ((const float *)p)[i] : dt == SF_F16 ? (float)((const f16 *)p)[i] : sf_bf16_to_f32(((const uint16_t *)p)[i]);
}

template <int CTRL>
__device__ __forceinline__ double q4_dpp(double v) {
  const uint64_t u = sf_bitcast<uint64_t>(v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, 0xF, 0xF, false);
  return sf_bitcast<double>((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double q4_swap16(double v) {
  const uint64_t u = sf_bitcast<uint64_t>(v);
  return sf_bitcast<double>((uint64_t)(uint32_t)__shfl_xor((int)(u >> 32), 16, 64) << 32 | (uint32_t)__shfl_xor((int)(uint32_t)u, 16, 64));
}
// f over aligned groups of n lanes (n = 2 .. 32, uniform); every lane gets the result.
template <class F>
__device__ __forceinline__ double q4_over(double v, int n, F f) {
  v = f(v, q4_dpp<0xB1>(v));
  if (n > 2) v = f(v, q4_dpp<0x4E>(v));
  if (n > 4) v = f(v, q4_dpp<0x141>(v));
  if (n > 8) v = f(v, q4_dpp<0x140>(v));
  if (n > 16) v = f(v, q4_swap16(v));
  return v;
}

// PAIR8: a lane's partners in the rotation are 8 neighbouring dims of the head (or its own).
template <int DT, bool PAIR8>
__global__ void __launch_bounds__(kQ4Threads)
k_kv_q4_append(Q4Append a, RotaryPos pos, const double *__restrict__ inv_freq) {
  extern __shared__ __attribute__((aligned(16))) double q4_smem[];
  const int D = a.D, P = a.P, heads = a.H + 2 * a.KVH, hb = kQ4Threads >> a.lanes_log2, L = 1 << a.lanes_log2;
  double *const ws = q4_smem;                                  // [2][D] norm weights
  double2 *const cs = (double2 *)(q4_smem + (a.qw || a.kw ? 2 * D : 0));  // [rows][P]
  const int first = blockIdx.x * hb, last = min(first + hb, a.n_heads) - 1;
  const int slot = threadIdx.x >> a.lanes_log2, i = threadIdx.x & (L - 1);
  const int row0 = first / heads, rows = last / heads - row0 + 1;
  const int e = min(first + slot, last), row = e / heads, hh = e - row * heads, b = row / a.T, t = row - b * a.T;
  const bool live = first + slot <= last && 8 * i < D, is_q = hh < a.H, is_v = hh >= a.H + a.KVH;
  const Q4Rows &x = is_q ? a.q : is_v ? a.v : a.k;
  const int h = is_q ? hh : is_v ? hh - a.H - a.KVH : hh - a.H;
  const size_t src = (size_t)(b * x.sb + t * x.st + h * x.sh);
  const int d0 = 8 * min(i, D / 8 - 1);
  const void *const w = is_q ? a.qw : is_v ? nullptr : a.kw;
  const int wo = is_q ? 0 : D;
  // dims d0 .. + 7 and the dims that turn with them
  float own[8], oth[8];
  const bool turns = !is_v && (PAIR8 ? d0 < 2 * P : true);
  auto partner = [&](int d) { return d >= 2 * P ? d : a.interleaved ? d ^ 1 : d < P ? d + P : d - P; };
  sf_load8_as_f32<DT>(x.x, src + d0, own);
  if constexpr (PAIR8) {
    if (!a.interleaved && turns) sf_load8_as_f32<DT>(x.x, src + partner(d0), oth);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) oth[j] = is_v ? 0.f : sf_load_as_f32<DT>(x.x, src + partner(d0 + j));
  }
  if (a.qw || a.kw)
    for (int d = threadIdx.x; d < 2 * D; d += kQ4Threads) {
      const void *p = d < D ? a.qw : a.kw;
      ws[d] = p ? q4_load(p, a.w_dtype, d < D ? d : d - D) : 1.0;
    }
  for (int n = threadIdx.x; n < rows * P; n += kQ4Threads) {
    const int r = n / P, rw = row0 + r, rb = rw / a.T;
    double c, s;
    rotary_sincos<true>((double)pos.at(rb, rw - rb * a.T) * inv_freq[n - r * P], c, s);
    cs[n] = double2{a.scale * c, a.scale * s};
  }
  __syncthreads();

  double y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = own[j];
  double r = 1.0;
  if (a.qw || a.kw) {
    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fma(y[j], y[j], ss);
    ss = q4_over(8 * i < D ? ss : 0.0, L, [](double p, double q) { return p + q; });
    if (w) {
      r = 1.0 / sqrt(ss / D + (double)a.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = y[j] * r * ws[wo + d0 + j];
    }
  }
  if (turns) {
    double z[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (PAIR8 && a.interleaved) {
        z[j] = y[j ^ 1];
      } else {
        z[j] = oth[j];
        if (w) z[j] = z[j] * r * ws[wo + partner(d0 + j)];
      }
    }
    const double2 *c = cs + (row - row0) * P;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = d0 + j;
      if (!PAIR8 && d >= 2 * P) continue;
      const bool second = a.interleaved ? d & 1 : d >= P;
      const double2 cj = c[a.interleaved ? d >> 1 : second ? d - P : d];
      y[j] = fma(y[j], cj.x, second ? z[j] * cj.y : -z[j] * cj.y);
    }
  }
  if (is_q) {
    if (!live) return;
    const size_t o = ((size_t)row * a.H + h) * D + d0;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (float)y[j];
    if (a.q_dtype == SF_F32) {
      float4_t *p = (float4_t *)((float *)a.q_out + o);
      p[0] = float4_t{f[0], f[1], f[2], f[3]};
      p[1] = float4_t{f[4], f[5], f[6], f[7]};
    } else {
      uint32_t u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = a.q_dtype == SF_BF16 ? sf_f32_to_bf16(f[j]) : sf_bitcast<uint16_t>((f16)sf_opaque(f[j]));
      *(u32x4 *)((uint16_t *)a.q_out + o) = u32x4{u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16};
    }
    return;
  }
  // k or v: the group's range over its lanes (the head's lanes past its dims stand aside)
  const bool in = 8 * i < D;
  double lo = y[0], hi = y[0];
  bool bad = false;  // a value that is not finite: the group reads back as NaN
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    lo = fmin(lo, y[j]);
    hi = fmax(hi, y[j]);
    bad = bad || !(fabs(y[j]) < INFINITY);
  }
  const int GL = a.g == D ? L : a.g / 8;
  lo = q4_over(in ? lo : (double)INFINITY, GL, [](double p, double q) { return fmin(p, q); });
  hi = q4_over(in ? hi : -(double)INFINITY, GL, [](double p, double q) { return fmax(p, q); });
  bad = q4_over(in && bad ? 1.0 : 0.0, GL, [](double p, double q) { return fmax(p, q); }) != 0.0;
  // (to fp32 first, as a conversion through fp32 would have it; held within fp16's range)
  const float lof = sf_opaque((float)lo), stf = sf_opaque((float)((hi - lo) / 15.0));
  f16 m16 = (f16)fminf(fmaxf(lof, -65504.f), 65504.f), s16 = (f16)fminf(stf, 65504.f);
  const double m = (double)m16, s = (double)s16, inv = s > 0.0 ? 1.0 / s : 0.0, half = 0.5 * s;
  uint32_t codes = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const double d = y[j] - m;
    double c = fmin(fmax(rint(d * inv), 0.0), 15.0);
    // the remainder says whether a border, or a tie that belongs to the even code, was missed
    const double rem = fma(-c, s, d);
    const bool odd = (int)c & 1;
    c += (rem > half || (rem == half && odd)) && s > 0.0 ? 1.0 : 0.0;
    c -= (rem < -half || (rem == -half && odd)) && s > 0.0 ? 1.0 : 0.0;
    codes |= (uint32_t)fmin(fmax(c, 0.0), 15.0) << (4 * j);
  }
  const long long len = a.lengths ? a.lengths[b] : a.start, at = len + t;
  if (!live || len < 0 || at >= a.T_cap) return;  // no such slot: nothing is written
  const size_t crow = ((size_t)b * a.KVH + h) * a.T_cap + (size_t)at;
  *(uint32_t *)((is_v ? a.vc : a.kc) + crow * (D / 2) + d0 / 2) = bad ? 0u : codes;
  if (d0 % a.g == 0) {
    const uint32_t word = sf_bitcast<uint16_t>(s16) | (uint32_t)sf_bitcast<uint16_t>(m16) << 16;
    (is_v ? a.vp : a.kp)[crow * (D / a.g) + d0 / a.g] = bad ? 0x7e007e00u : word;
  }
}

// Eight values a thread: a word of codes, 16 or 32 bytes out.
template <int DT>
__global__ void __launch_bounds__(kQ4Threads)
k_kv_q4_dequant(const uint8_t *__restrict__ codes, const uint32_t *__restrict__ params, void *__restrict__ out, int KVH,
                int T, int D, int g, long long cb, long long ch, long long ct, long long pb, long long ph, long long pt,
                long long n) {
  const long long e = (long long)blockIdx.x * kQ4Threads + threadIdx.x;
  if (e >= n) return;
  const int oct = D / 8;
  const long long row = e / oct;
  const int i = (int)(e - row * oct), t = (int)(row % T);
  const long long bh = row / T;
  const int h = (int)(bh % KVH);
  const long long b = bh / KVH;
  const uint32_t c = *(const uint32_t *)(codes + b * cb + h * ch + t * ct + 4 * i);
  const uint32_t w = params[b * pb + h * ph + t * pt + 8 * i / g];
  const float s = (float)sf_bitcast<f16>((uint16_t)(w & 0xffffu)), m = (float)sf_bitcast<f16>((uint16_t)(w >> 16));
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = fmaf((float)(c >> (4 * j) & 15u), s, m);
  if constexpr (DT == SF_F32) {
    float4_t *p = (float4_t *)((float *)out + 8 * e);
    p[0] = float4_t{f[0], f[1], f[2], f[3]};
    p[1] = float4_t{f[4], f[5], f[6], f[7]};
  } else {
    Vec<DT> v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v.v[j] = f[j];
    ((u32x4 *)out)[e] = v.pack();
  }
}

}  // namespace

int sf_q4_cache_check(int D, int g) {
  SF_REQUIRE(D > 0 && g > 0 && D % g == 0, SF_EINVAL, "head_dim=%d must be divisible by group=%d", D, g);
  SF_REQUIRE(D <= kQ4MaxD, SF_EINVAL, "head_dim=%d exceeds kernel's compile-time max %d", D, kQ4MaxD);
  SF_REQUIRE(D % 16 == 0, SF_EUNSUPPORTED, "head_dim=%d: need a multiple of 16", D);
  SF_REQUIRE(g == D || g == 32 || g == 64 || g == 128, SF_EUNSUPPORTED,
             "group=%d: need 32, 64, 128 or the whole head of %d", g, D);
  return SF_OK;
}

extern "C" int sf_kv_q4_append(const void *q, const void *k, const void *v, int in_dtype, const long long *strides,
                               const void *q_weight, const void *k_weight, int weight_dtype, float eps,
                               const void *positions, int pos_i64, int pos_per_seq, const double *inv_freq,
                               int rot_pairs, float scale, int interleaved, void *q_out, int q_dtype, uint8_t *k_codes,
                               void *k_params, uint8_t *v_codes, void *v_params, int group, const int32_t *lengths,
                               int start, int B, int T, int H, int KVH, int D, int T_cap, void *stream) {
  SF_REQUIRE(B >= 0 && T >= 0 && H >= 0 && KVH > 0, SF_EINVAL, "invalid KV shape B=%d T=%d H=%d KVH=%d", B, T, H, KVH);
  if (int rc = sf_q4_cache_check(D, group)) return rc;
  SF_REQUIRE(rot_pairs >= 0 && 2LL * rot_pairs <= D, SF_EINVAL, "%d rotated pairs in a head of %d", rot_pairs, D);
  SF_REQUIRE(in_dtype >= SF_F32 && in_dtype <= SF_BF16 && (H == 0 || (q_dtype >= SF_F32 && q_dtype <= SF_BF16)) &&
                 ((!q_weight && !k_weight) || (weight_dtype >= SF_F32 && weight_dtype <= SF_BF16)),
             SF_EINVAL, "bad input / q / weight dtype");
  SF_REQUIRE(T_cap > 0 && (lengths || (start >= 0 && (long long)start + T <= T_cap)), SF_EINVAL,
             "KV cache overflow: %d + %d > capacity %d", start, T, T_cap);
  const long long n_heads = (long long)B * T * (H + 2LL * KVH);
  SF_REQUIRE(n_heads <= 0x7fffffffLL - 65536, SF_EINVAL, "%d x %d rows of %d heads exceed the grid", B, T, H + 2 * KVH);
  if (n_heads == 0) return SF_OK;
  SF_REQUIRE(k && v && strides && (H == 0 || (q && q_out)) && k_codes && k_params && v_codes && v_params &&
                 (rot_pairs == 0 || (positions && inv_freq)),
             SF_EINVAL, "null pointer argument");
  const long long *s = strides;
  bool whole = (((uintptr_t)k | (uintptr_t)v | (H ? (uintptr_t)q | (uintptr_t)q_out : 0)) & 15) == 0;
  for (int n = H ? 0 : 3; n < 9; ++n) whole = whole && s[n] % 8 == 0;
  SF_REQUIRE(whole, SF_EINVAL, "q, k, v and q_out must start on 16 bytes and have strides of whole 8 elements");
  SF_REQUIRE((((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_params | (uintptr_t)v_params) & 15) == 0, SF_EINVAL,
             "cache buffers must be 16-byte aligned");
  Q4Append a = {{q, s[0], s[1], s[2]}, {k, s[3], s[4], s[5]}, {v, s[6], s[7], s[8]}, q_weight, k_weight, q_out, k_codes,
                v_codes, (uint32_t *)k_params, (uint32_t *)v_params, lengths, start, q_dtype, weight_dtype, H, KVH, D,
                group, T, T_cap, rot_pairs, interleaved, 1, (int)n_heads, eps, scale};
  while ((8 << a.lanes_log2) < D) ++a.lanes_log2;
  const int hb = kQ4Threads >> a.lanes_log2, heads = H + 2 * KVH, rows = (hb + heads - 2) / heads + 1;
  const size_t lds = (size_t)(q_weight || k_weight ? 2 * D : 0) * 8 + (size_t)rows * rot_pairs * 16 + 16;
  const RotaryPos pos = {positions, pos_i64, pos_per_seq ? T : 0};
  const unsigned grid = (unsigned)((n_heads + hb - 1) / hb);
  const bool pair8 = (interleaved ? 2 * rot_pairs : rot_pairs) % 8 == 0;
  hipStream_t st = (hipStream_t)stream;
#define SF_Q4A(DT)                                                                            \
  do {                                                                                        \
    if (pair8) k_kv_q4_append<DT, true><<<grid, kQ4Threads, lds, st>>>(a, pos, inv_freq);     \
    else k_kv_q4_append<DT, false><<<grid, kQ4Threads, lds, st>>>(a, pos, inv_freq);          \
  } while (0)
  if (in_dtype == SF_F32) SF_Q4A(SF_F32);
  else if (in_dtype == SF_F16) SF_Q4A(SF_F16);
  else SF_Q4A(SF_BF16);
#undef SF_Q4A
  return sf_check_launch("sf_kv_q4_append");
}

extern "C" int sf_kv_q4_dequant(const uint8_t *codes, const void *params, void *out, int out_dtype, int group,
                                const long long *strides, int B, int KVH, int T, int D, void *stream) {
  SF_REQUIRE(B >= 0 && KVH >= 0 && T >= 0, SF_EINVAL, "invalid KV shape B=%d KVH=%d T=%d", B, KVH, T);
  if (int rc = sf_q4_cache_check(D, group)) return rc;
  SF_REQUIRE(out_dtype >= SF_F32 && out_dtype <= SF_BF16, SF_EINVAL, "bad out dtype %d", out_dtype);
  const long long rows = (long long)B * KVH;
  if (rows == 0 || T == 0) return SF_OK;
  SF_REQUIRE(codes && params && out && strides, SF_EINVAL, "null pointer argument");
  SF_REQUIRE(((uintptr_t)codes & 3) == 0 && ((uintptr_t)params & 3) == 0 && ((uintptr_t)out & 15) == 0 &&
                 strides[0] % 4 == 0 && strides[1] % 4 == 0 && strides[2] % 4 == 0 && strides[3] % 2 == 0 &&
                 strides[4] % 2 == 0 && strides[5] % 2 == 0,
             SF_EINVAL, "codes and params must have rows on 4 bytes, out must be 16-byte aligned");
  SF_REQUIRE(rows <= 0x7fffffffLL * 256 / T / (D / 8), SF_EINVAL, "B=%d KVH=%d T=%d exceed the grid", B, KVH, T);
  const long long n = rows * T * (D / 8);
  const unsigned grid = (unsigned)((n + kQ4Threads - 1) / kQ4Threads);
  hipStream_t st = (hipStream_t)stream;
#define SF_Q4D(DT)                                                                                                     \
  k_kv_q4_dequant<DT><<<grid, kQ4Threads, 0, st>>>(codes, (const uint32_t *)params, out, KVH, T, D, group, strides[0], \
                                                   strides[1], strides[2], strides[3] / 2, strides[4] / 2, strides[5] / 2, n)
  if (out_dtype == SF_F32) SF_Q4D(SF_F32);
  else if (out_dtype == SF_F16) SF_Q4D(SF_F16);
  else SF_Q4D(SF_BF16);
#undef SF_Q4D
  return sf_check_launch("sf_kv_q4_dequant");
}
