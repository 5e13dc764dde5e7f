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

// cos and sin of pos * f times scale, in fp32: the angle less its nearest multiple of
// pi / 2 (in two parts, so that what is left is exact to 2^-53 of the angle), then the
// series of sine and cosine on [-pi/4, pi/4] in 64 bits, to r^11 and r^12: 7e-12 at most,
// so c and s are the nearest fp32 values but for one in some thousands. Some 30 64-bit
// operations a pair (the library's sincos takes a longer reduction for far positions:
// 16 tokens near 500000 10.6 us, this 3.0).
__device__ __forceinline__ float2_t rotary_cs(long long pos, double f, float scale) {
  const double a = (double)pos * f, n = rint(a * 0.63661977236758134308);
  const double r = fma(-n, 6.123233995736766036e-17, fma(-n, 1.57079632679489661923, a)), z = r * r;
  double s = -1.0 / 39916800, c = 1.0 / 479001600;
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
  return float2_t{(float)(scale * (q == 1 || q == 2 ? -cq : cq)), (float)(scale * (q & 2 ? -sq : sq))};
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
constexpr int kRotTable = 1024;  // cos / sin pairs of a workgroup's rows

// How a workgroup's work is cut: `rows` rows of `items` items, `per` a head.
struct RotaryCut {
  int rows, items, per, n_rows;
  uint32_t inv_items, inv_per;  // ceil(2^32 / .), exact below 2^16 items; 0 stands for a division by 1
};
__device__ __forceinline__ int div_by(int e, uint32_t inv) { return inv ? (int)__umulhi((uint32_t)e, inv) : e; }

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
        w[j] = sf_f32_to_bf16(v[2 * j]) | (uint32_t)sf_f32_to_bf16(v[2 * j + 1]) << 16;
      }
    }
    return w;
  }
};

// VEC: an item is 16 bytes of a head (and, half layout, the 16 bytes P dims further that
// turn with them), loaded before the workgroup computes its cos / sin table. Else an item
// is one pair, or one dim past the rotated part. Bound by the memory stream; rows of a
// workgroup share nothing, several are taken together only to fill its threads.
// 8191 rows of 32 / 8 heads of 128, bf16 (168 MB), us a call in a row of them: single dims and
// the library's sincos 90, this 34.7 (a 1 GiB copy's rate would take 33). Two, four items a thread
// take 38.2, 40.1, and stores past the caches end the kernel sooner, but not the call.
template <int DT, bool VEC, bool INTER>
__global__ void __launch_bounds__(kRotThreads)
k_rotary(RotaryRows q, RotaryRows k, RotaryPos pos, const double *__restrict__ inv_freq, int P, float scale, int T,
         int D, RotaryCut cut) {
  constexpr int E = Vec<DT>::E, kItems = 1;  // a thread's items per round
  __shared__ float2_t cs[kRotTable];
  const int row0 = blockIdx.x * cut.rows, rows = min(cut.rows, cut.n_rows - row0);
  const int n = rows * cut.items, turned = VEC ? (INTER ? 2 * P / E : P / E) : P;
  struct Item {
    const void *in;
    void *out;
    size_t src, dst;
    int i, tab;  // item of its head; its row's place in the table
  };
  auto item = [&](int e) {
    const int r = div_by(e, cut.inv_items), eh = e - r * cut.items;
    const int hh = div_by(eh, cut.inv_per), row = row0 + r, b = row / T, t = row - b * T;
    const RotaryRows &x = hh < q.heads ? q : k;
    const int h = hh < q.heads ? hh : hh - q.heads;
    return Item{x.in, x.out, (size_t)(b * x.ib + t * x.it + h * x.ih), (size_t)(b * x.ob + t * x.ot + h * x.oh),
                eh - hh * cut.per, r * P};
  };
  bool have_cs = false;
  for (int e0 = threadIdx.x; e0 - (int)threadIdx.x < n; e0 += kItems * kRotThreads) {
    Item it[kItems];
    u32x4 lo[kItems], hi[kItems];
    if constexpr (VEC) {
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        const int e = e0 + u * kRotThreads;
        if (e >= n) continue;
        it[u] = item(e);
        const int i = it[u].i, d = i < turned ? i * E : 2 * P + (i - turned) * E;
        constexpr int sz = DT == SF_F32 ? 4 : 2;
        lo[u] = *(const u32x4 *)((const char *)it[u].in + (it[u].src + d) * sz);
        if (!INTER && i < turned) hi[u] = *(const u32x4 *)((const char *)it[u].in + (it[u].src + d + P) * sz);
      }
    }
    if (!have_cs) {
      for (int i = threadIdx.x; i < rows * P; i += kRotThreads) {
        const int r = i / P, row = row0 + r, b = row / T;
        cs[i] = rotary_cs(pos.at(b, row - b * T), inv_freq[i - r * P], scale);
      }
      __syncthreads();
      have_cs = true;
    }
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const int e = e0 + u * kRotThreads;
      if (e >= n) continue;
      if constexpr (VEC) {
        const int i = it[u].i, d = i < turned ? i * E : 2 * P + (i - turned) * E;
        constexpr int sz = DT == SF_F32 ? 4 : 2;
        char *o = (char *)it[u].out + (it[u].dst + d) * sz;
        if (i < turned) {
          Vec<DT> a, c;
          a.load(lo[u]);
          if constexpr (INTER) {
#pragma unroll
            for (int j = 0; j < E; j += 2) {
              const float2_t y = turn(a.v[j], a.v[j + 1], cs[it[u].tab + (i * E + j) / 2]);
              a.v[j] = y.x;
              a.v[j + 1] = y.y;
            }
          } else {
            c.load(hi[u]);
#pragma unroll
            for (int j = 0; j < E; ++j) {
              const float2_t y = turn(a.v[j], c.v[j], cs[it[u].tab + i * E + j]);
              a.v[j] = y.x;
              c.v[j] = y.y;
            }
            *(u32x4 *)(o + P * sz) = c.pack();
          }
          lo[u] = a.pack();
        }
        *(u32x4 *)o = lo[u];
      } else {
        const Item x = item(e);
        if (x.i < P) {
          const int d1 = INTER ? 2 * x.i : x.i, d2 = INTER ? d1 + 1 : x.i + P;
          const float2_t y = turn(sf_load_as_f32<DT>(x.in, x.src + d1), sf_load_as_f32<DT>(x.in, x.src + d2),
                                  cs[x.tab + x.i]);
          sf_store_from_f32<DT>(x.out, x.dst + d1, sf_opaque(y.x));
          sf_store_from_f32<DT>(x.out, x.dst + d2, sf_opaque(y.y));
        } else {
          const int d = P + x.i;
          sf_store_from_f32<DT>(x.out, x.dst + d, sf_load_as_f32<DT>(x.in, x.src + d));
        }
      }
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
  const int len = a.lengths ? a.lengths[b] : a.start;
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
  // 16 bytes at a time where every head starts on 16 bytes and its parts are whole vectors
  const int E = dtype == SF_F32 ? 4 : 8, rest = D - 2 * rot_pairs;
  bool vec = rest % E == 0 && (interleaved ? 2 * rot_pairs : rot_pairs) % E == 0 &&
             (((uintptr_t)q | (uintptr_t)q_out | (KVH ? (uintptr_t)k | (uintptr_t)k_out : 0)) & 15) == 0;
  for (int i = 0; i < (KVH ? 12 : 6); ++i) vec = vec && s[i] % E == 0;
  RotaryCut cut;
  cut.per = vec ? (interleaved ? 2 * rot_pairs : rot_pairs) / E + rest / E : rot_pairs + rest;
  SF_REQUIRE((long long)(H + KVH) * cut.per < 65536, SF_EUNSUPPORTED, "%d heads of %d dims a row: too wide", H + KVH, D);
  cut.items = (H + KVH) * cut.per;
  cut.n_rows = B * T;
  // rows a workgroup: one item a thread, while that leaves two workgroups a CU
  int rows = kRotThreads / cut.items;
  if (rows > cut.n_rows / 512) rows = cut.n_rows / 512;
  if (rows > kRotTable / rot_pairs) rows = kRotTable / rot_pairs;
  if (rows > 65535 / cut.items) rows = 65535 / cut.items;
  cut.rows = rows < 1 ? 1 : rows;
  cut.inv_items = cut.items == 1 ? 0 : (uint32_t)(((1ull << 32) + cut.items - 1) / cut.items);
  cut.inv_per = cut.per == 1 ? 0 : (uint32_t)(((1ull << 32) + cut.per - 1) / cut.per);
  const unsigned grid = (unsigned)((cut.n_rows + cut.rows - 1) / cut.rows);
#define SF_ROT(DT, V, I) \
  k_rotary<DT, V, I><<<grid, kRotThreads, 0, st>>>(rq, rk, pos, inv_freq, rot_pairs, scale, T, D, cut)
#define SF_ROT_D(DT)                         \
  do {                                       \
    if (vec && interleaved) SF_ROT(DT, true, true);   \
    else if (vec) SF_ROT(DT, true, false);   \
    else if (interleaved) SF_ROT(DT, false, true);    \
    else SF_ROT(DT, false, false);           \
  } while (0)
  if (dtype == SF_F32) SF_ROT_D(SF_F32);
  else if (dtype == SF_F16) SF_ROT_D(SF_F16);
  else SF_ROT_D(SF_BF16);
#undef SF_ROT_D
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
