// kv_q4.hip — a KV cache held in 4 bits: append and reading back (gfx950).
//
// A head's D dims of a token are cut into groups of g; a group holds
//   m = f16(min x),  s = f16((max x - min x) / 15),
//   code = clip(rint((x - m) / s), 0, 15)  (0 where s is 0),  x ~ m + s code,
// s and m held at the ends of fp16's range;
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
  int start, q_dtype, w_dtype, H, KVH, D, g, g_log2, groups, T, T_cap, P, lanes_log2, n_heads, chunks;
  uint32_t inv_heads, inv_T, inv_P;  // for div_by
  float eps, scale;
  double inv_D;
};

__device__ __forceinline__ double q4_load(const void *p, int dt, size_t i) {
  return dt == SF_F32 ? ((const float *)p)[i] : dt == SF_F16 ? (float)((const f16 *)p)[i] : sf_bf16_to_f32(((const uint16_t *)p)[i]);
}

// A whole number as an int, held within its range (the hardware's conversion; NaN as 0, which
// a plain cast leaves open).
__device__ __forceinline__ int q4_int(double v) {
  int r;
  asm("v_cvt_i32_f64 %0, %1" : "=v"(r) : "v"(v));
  return r;
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
template <int CTRL>
__device__ __forceinline__ float q4_dpp(float v) { return sf_dpp<CTRL>(v); }
__device__ __forceinline__ float q4_swap16(float v) { return __shfl_xor(v, 16, 64); }
// f over aligned groups of n lanes (n = 2 .. 32, uniform); every lane gets the result.
template <class V, class F>
__device__ __forceinline__ V q4_over(V v, int n, F f) {
  v = f(v, q4_dpp<0xB1>(v));
  if (n > 2) v = f(v, q4_dpp<0x4E>(v));
  if (n > 4) v = f(v, q4_dpp<0x141>(v));
  if (n > 8) v = f(v, q4_dpp<0x140>(v));
  if (n > 16) v = f(v, q4_swap16(v));
  return v;
}

// PAIR8: a lane's partners in the rotation are 8 neighbouring dims of the head (INTER: its own).
// Bound by vector instructions: 4095 rows of 32 / 8 heads of 128, bf16, groups of 64, normed and
// turned, 88 MB (17 us at a copy's rate) in 42 us, vector instructions in 85% of the SIMDs' time: 60.8 with divisions for the head, the row, the
// scale's inverse and the root and every code's remainder settled, 53 with the tables in the
// dims' order (a head's lanes on the same banks).
template <int DT, bool PAIR8, bool INTER>
__global__ void __launch_bounds__(kQ4Threads)
k_kv_q4_append(Q4Append a, RotaryPos pos, const double *__restrict__ inv_freq) {
  extern __shared__ __attribute__((aligned(16))) double q4_smem[];
  const int D = a.D, P = a.P, heads = a.H + 2 * a.KVH, hb = kQ4Threads >> a.lanes_log2, L = 1 << a.lanes_log2;
  double *const ws = q4_smem;                                  // [2][D] norm weights
  double2 *const cs = (double2 *)(q4_smem + (a.qw || a.kw ? 2 * D : 0));  // [rows][P]
  // The workgroup's first head, row and token by (uniform) divisions, a lane's by what it is past
  // them; a.chunks times hb heads, the next ones' rows loaded during the last ones' arithmetic.
  const int first = blockIdx.x * hb * a.chunks, row0 = first / heads, off0 = first - row0 * heads;
  const int b0 = row0 / a.T, t0 = row0 - b0 * a.T;
  const int count = min(hb * a.chunks, a.n_heads - first);
  const int slot = threadIdx.x >> a.lanes_log2, i = threadIdx.x & (L - 1);
  const int rows = div_by(off0 + count - 1, a.inv_heads) + 1;
  // (a row's token: rows of a workgroup are few, so that past 2^15 tokens one sequence at most ends among them)
  auto token = [&](int r, int &b, int &t) {
    const int x = t0 + r, n = a.T < 32768 ? div_by(x, a.inv_T) : x >= a.T;
    b = b0 + n;
    t = x - n * a.T;
  };
  const bool in = 8 * i < D, normed = a.qw || a.kw;
  const int d0 = 8 * min(i, D / 8 - 1);
  const bool second = d0 >= P;
  // a lane's j-th weight and pair lie beside its neighbours' j-th: 8 dims a lane in order would have
  // every lane of a head read the same banks
  const int oct = D / 8, pairs = INTER ? P / 4 : P / 8;
  auto weight_at = [&](int d) { return (d & 7) * oct + (d >> 3); };
  auto pair_at = [&](int p) { return !PAIR8 ? p : INTER ? (p & 3) * pairs + (p >> 2) : (p & 7) * pairs + (p >> 3); };
  auto partner = [&](int d) { return d >= 2 * P ? d : INTER ? d ^ 1 : d < P ? d + P : d - P; };
  const int p0 = second ? d0 - P : d0 + P;  // (PAIR8, half layout)
  // a lane's head, and its dims d0 .. + 7 and those that turn with them
  struct Head {
    int dr, b, t, h;
    bool is_q, is_v, live;
    float own[8], oth[8];
  };
  auto take = [&](int u, Head &x) {
    const int past = off0 + min(u * hb + slot, count - 1);
    x.dr = div_by(past, a.inv_heads);
    const int hh = past - x.dr * heads;
    token(x.dr, x.b, x.t);
    x.live = u * hb + slot < count && in;
    x.is_q = hh < a.H;
    x.is_v = hh >= a.H + a.KVH;
    x.h = x.is_q ? hh : x.is_v ? hh - a.H - a.KVH : hh - a.H;
    const Q4Rows &s = x.is_q ? a.q : x.is_v ? a.v : a.k;
    const size_t src = (size_t)(x.b * s.sb + x.t * s.st + x.h * s.sh);
    sf_load8_as_f32<DT>(s.x, src + d0, x.own);
    if constexpr (!PAIR8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x.oth[j] = x.is_v ? 0.f : sf_load_as_f32<DT>(s.x, src + partner(d0 + j));
    } else if constexpr (!INTER) {
      if (!x.is_v && d0 < 2 * P) sf_load8_as_f32<DT>(s.x, src + p0, x.oth);
    }
  };
  Head nxt;
  take(0, nxt);
  if (normed)
    for (int d = threadIdx.x; d < 2 * D; d += kQ4Threads) {
      const void *p = d < D ? a.qw : a.kw;
      ws[d < D ? weight_at(d) : D + weight_at(d - D)] = p ? q4_load(p, a.w_dtype, d < D ? d : d - D) : 1.0;
    }
  if (off0 < a.H + a.KVH || rows > 1)  // (v's heads alone need none)
    for (int n = threadIdx.x; n < rows * P; n += kQ4Threads) {
      const int r = div_by(n, a.inv_P), pr = n - r * P;
      int rb, rt;
      token(r, rb, rt);
      double c, s;
      rotary_sincos<true>((double)pos.at(rb, rt) * inv_freq[pr], c, s);
      cs[r * P + pair_at(pr)] = double2{a.scale * c, a.scale * s};
    }
  __syncthreads();

#pragma unroll 1
  for (int u = 0; u * hb < count; ++u) {
    const Head x = nxt;
    if ((u + 1) * hb < count) take(u + 1, nxt);
    const int b = x.b, t = x.t, h = x.h;
    const bool turns = !x.is_v && (PAIR8 ? d0 < 2 * P : true);
    const void *const w = x.is_q ? a.qw : x.is_v ? nullptr : a.kw;
    const double *const wo = ws + (x.is_q ? 0 : D);
    double y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = x.own[j];
    double r = 1.0;
    if (normed) {
      double ss = 0.0;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fma(y[j], y[j], ss);
      ss = q4_over(in ? ss : 0.0, L, [](double p, double q) { return p + q; });
      if (w) {
        // 1 / sqrt by the hardware's estimate and two steps of Newton's, to 2^-52
        const double v = ss * a.inv_D + (double)a.eps;
        r = __builtin_amdgcn_rsq(v);
        r = fma(fma(-v * r, r, 1.0), 0.5 * r, r);
        r = fma(fma(-v * r, r, 1.0), 0.5 * r, r);
        r = v == 0.0 ? (double)INFINITY : v == (double)INFINITY ? 0.0 : r;
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = y[j] * r * wo[j * oct + d0 / 8];
      }
    }
    if (turns) {
      const double2 *const c = cs + x.dr * P;
      if constexpr (PAIR8 && INTER) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const double2 cj = c[(j >> 1) * pairs + d0 / 8];
          const double lo = fma(y[j], cj.x, -y[j + 1] * cj.y), hi = fma(y[j + 1], cj.x, y[j] * cj.y);
          y[j] = lo;
          y[j + 1] = hi;
        }
      } else if constexpr (PAIR8) {
        const double turn = second ? r : -r;
        const double2 *const cp = c + (second ? d0 - P : d0) / 8;
        double z[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = x.oth[j] * turn;
        if (w) {
#pragma unroll
          for (int j = 0; j < 8; ++j) z[j] *= wo[j * oct + p0 / 8];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = fma(y[j], cp[j * pairs].x, z[j] * cp[j * pairs].y);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int d = d0 + j;
          if (d >= 2 * P) continue;
          double z = x.oth[j] * r;
          if (w) z *= wo[weight_at(partner(d))];
          const bool two = INTER ? d & 1 : d >= P;
          const double2 cj = c[INTER ? d >> 1 : two ? d - P : d];
          y[j] = fma(y[j], cj.x, two ? z * cj.y : -z * cj.y);
        }
      }
    }
    if (x.is_q) {
      if (!x.live) continue;
      const size_t o = (((size_t)b * a.T + t) * a.H + h) * D + d0;
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
      continue;
    }
    // k or v: the group's range over its lanes (the head's lanes past its dims stand aside)
    double lo = y[0], hi = y[0], all = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo = fmin(lo, y[j]);
      hi = fmax(hi, y[j]);
      all = fma(y[j], 0.0, all);  // NaN where a value is not finite: the group reads back as NaN
    }
    const int GL = a.g == D ? L : a.g / 8;
    lo = q4_over(in ? lo : (double)INFINITY, GL, [](double p, double q) { return fmin(p, q); });
    hi = q4_over(in ? hi : -(double)INFINITY, GL, [](double p, double q) { return fmax(p, q); });
    const bool bad = q4_over(in && all != 0.0 ? 1.f : 0.f, GL, [](float p, float q) { return fmaxf(p, q); }) != 0.f;
    // (to fp32 first, as a conversion through fp32 would have it; held within fp16's range. A
    // product with 1 / 15 is the quotient but for its last place in 64 bits, which fp32 drops.)
    const float lof = sf_opaque((float)lo), stf = sf_opaque((float)((hi - lo) * (1.0 / 15.0)));
    f16 m16 = (f16)fminf(fmaxf(lof, -65504.f), 65504.f), s16 = (f16)fminf(stf, 65504.f);
    const double m = (double)m16, s = (double)s16, half = 0.5 * s;
    const double inv = s > 0.0 ? __builtin_amdgcn_rcp(s) : 0.0;  // (an estimate: the remainders tell)
    double c[8];
    bool off = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double d = y[j] - m;
      c[j] = rint(d * inv);
      off = off || fabs(fma(-c[j], s, d)) >= half;
    }
    if (__any(off)) {  // a border, or a tie, which belongs to the even code
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const double rem = fma(-c[j], s, y[j] - m), odd = c[j] - 2.0 * floor(0.5 * c[j]);
        if (s > 0.0) c[j] += rem > half || (rem == half && odd != 0.0) ? 1.0 : rem < -half || (rem == -half && odd != 0.0) ? -1.0 : 0.0;
      }
    }
    uint32_t codes = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) codes |= (uint32_t)min(max(q4_int(c[j]), 0), 15) << (4 * j);
    const long long len = a.lengths ? a.lengths[b] : a.start, at = len + t;
    if (!x.live || len < 0 || at >= a.T_cap) continue;  // no such slot: nothing is written
    const size_t crow = ((size_t)b * a.KVH + h) * a.T_cap + (size_t)at;
    *(uint32_t *)((x.is_v ? a.vc : a.kc) + crow * (D / 2) + d0 / 2) = bad ? 0u : codes;
    const int gi = a.g == D ? 0 : d0 >> a.g_log2;
    if (d0 == gi * a.g) {
      const uint32_t word = sf_bitcast<uint16_t>(s16) | (uint32_t)sf_bitcast<uint16_t>(m16) << 16;
      (x.is_v ? a.vp : a.kp)[crow * a.groups + gi] = bad ? 0x7e007e00u : word;
    }
  }
}

// Eight values a thread: a word of codes, 16 or 32 bytes out. `blocks` workgroups a head. 4095 slots
// of 8 heads of 128 to fp32 (19 MB) 6.3 us traced: latency around 3.7 at a copy's rate.
template <int DT>
__global__ void __launch_bounds__(kQ4Threads)
k_kv_q4_dequant(const uint8_t *__restrict__ codes, const uint32_t *__restrict__ params, void *__restrict__ out, int KVH,
                int T, int D, int g_log2, int groups, long long cb, long long ch, long long ct, long long pb, long long ph,
                long long pt, unsigned blocks, uint32_t inv_oct) {
  // (uniform divisions, a lane's by what it is past them)
  const unsigned bh = blockIdx.x / blocks, s0 = (blockIdx.x - bh * blocks) * kQ4Threads, oct = D / 8;
  const unsigned b = bh / KVH, h = bh - b * KVH, t0 = s0 / oct, past = s0 - t0 * oct + threadIdx.x;
  const int dt = div_by(past, inv_oct), i = past - dt * oct;
  const long long t = (long long)t0 + dt;
  if (t >= T) return;
  const size_t e = ((size_t)bh * T + t) * oct + i;
  const uint32_t c = *(const uint32_t *)(codes + b * cb + h * ch + t * ct + 4 * i);
  const uint32_t w = params[b * pb + h * ph + t * pt + (groups == 1 ? 0 : 8 * i >> g_log2)];
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
  SF_REQUIRE(H <= 16384 && KVH <= 8192, SF_EUNSUPPORTED, "%d and %d heads: at most 16384 and 8192", H, KVH);
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
                group, 5, D / group, T, T_cap, rot_pairs, 1, (int)n_heads, 1, div_inv(H + 2 * KVH), div_inv(T),
                rot_pairs ? div_inv(rot_pairs) : 0, eps, scale, 1.0 / D};
  while ((1 << a.g_log2) < group) ++a.g_log2;
  while ((8 << a.lanes_log2) < D) ++a.lanes_log2;
  // Three times the heads that a workgroup's threads hold, where that leaves four workgroups a CU: its
  // weights and table serve as many (us a call, 4095 / 2048 / 1024 rows of the above: one 51.4 / 27.5 /
  // 16.6, two 44.8 / 24.7 / 15.8, three 42.0 / 23.2 / 14.6, four 42.2 / 25.1 / 15.4, six 42.3 / 24.0 / 17.7;
  // in a replayed graph at the border and at four times as many, one / three: 14 / 2 heads of 64 18.1 / 16.8 and 58.2 /
  // 48.1, 9 / 3 of 80 17.7 / 17.6 and 58.5 / 51.3, 16 / 4 of 256 16.7 / 14.1 and 53.4 / 40.9, 32 / 32 of 128 15.7 / 14.7
  // and 49.1 / 43.2; k and v alone, 4095 rows of 8 heads of 128, 16.3 / 16.7, 16000 rows 50.9 / 45.1).
  const int hb = kQ4Threads >> a.lanes_log2, heads = H + 2 * KVH;
  a.chunks = n_heads >= 3LL * hb * 1024 ? 3 : 1;
  const int rows = (hb * a.chunks + heads - 2) / heads + 1;
  const size_t lds = (size_t)(q_weight || k_weight ? 2 * D : 0) * 8 + (size_t)rows * rot_pairs * 16 + 16;
  const RotaryPos pos = {positions, pos_i64, pos_per_seq ? T : 0};
  const unsigned grid = (unsigned)((n_heads + hb * a.chunks - 1) / (hb * a.chunks));
  const bool pair8 = (interleaved ? 2 * rot_pairs : rot_pairs) % 8 == 0;
  hipStream_t st = (hipStream_t)stream;
#define SF_Q4A_I(DT, P8, I) k_kv_q4_append<DT, P8, I><<<grid, kQ4Threads, lds, st>>>(a, pos, inv_freq)
#define SF_Q4A(DT)                                                                            \
  do {                                                                                        \
    if (pair8 && interleaved) SF_Q4A_I(DT, true, true);                                       \
    else if (pair8) SF_Q4A_I(DT, true, false);                                                \
    else if (interleaved) SF_Q4A_I(DT, false, true);                                          \
    else SF_Q4A_I(DT, false, false);                                                          \
  } while (0)
  if (in_dtype == SF_F32) SF_Q4A(SF_F32);
  else if (in_dtype == SF_F16) SF_Q4A(SF_F16);
  else SF_Q4A(SF_BF16);
#undef SF_Q4A
#undef SF_Q4A_I
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
  const long long blocks = ((long long)T * (D / 8) + kQ4Threads - 1) / kQ4Threads;
  SF_REQUIRE(blocks <= 1 << 23 && rows <= 0x7fffffffLL / blocks, SF_EINVAL, "B=%d KVH=%d T=%d exceed the grid", B, KVH, T);
  const unsigned grid = (unsigned)(rows * blocks);
  int g_log2 = 0;
  while ((1 << g_log2) < group) ++g_log2;
  hipStream_t st = (hipStream_t)stream;
#define SF_Q4D(DT)                                                                                                     \
  k_kv_q4_dequant<DT><<<grid, kQ4Threads, 0, st>>>(codes, (const uint32_t *)params, out, KVH, T, D, g_log2, D / group, \
                                                   strides[0], strides[1], strides[2], strides[3] / 2, strides[4] / 2, \
                                                   strides[5] / 2, (unsigned)blocks, div_inv(D / 8))
  if (out_dtype == SF_F32) SF_Q4D(SF_F32);
  else if (out_dtype == SF_F16) SF_Q4D(SF_F16);
  else SF_Q4D(SF_BF16);
#undef SF_Q4D
  return sf_check_launch("sf_kv_q4_dequant");
}
