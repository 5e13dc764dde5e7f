// qk_norm.hip — queries and keys normed a head and rotated in one pass (gfx950).
//
// A head x of D dims, with r = 1 / sqrt(mean(x^2) + eps) and its side's weights w:
//   n = x r,  y = R(p) (n w),
// R(p) the rotation of rotary.hip (pairs turned at position p, cos and sin times scale,
// dims past them as they are). Backward, for the gradient gy of y:
//   g = R(p)^T gy,  dw = sum over rows and heads of g n,
//   dx = r (g w - n mean(g w n)).
// All in fp32 (the angle in 64 bits), one rounding to the output's type at the end.
//
//   sf_qk_norm_rotary            q (and k) rows, any strides, in place or not
//   sf_qk_norm_rotary_backward   dq, dk and both weights' gradients
//
// L lanes hold a head (the power of two that covers its items), an item being 16 bytes of
// it and, half layout, the 16 bytes P dims further that turn with them: one load of the
// row, the sum of squares over L lanes in registers, one store. Bound by the memory stream:
// 8191 rows of 32 / 8 heads of 128 in bf16 (168 MB) 30.6 us traced, 37.9 a call over memory that
// is not cached, where a copy's rate gives 32; 4084 rows with half of each head turned, pairs
// interleaved, forward 24.0 (84 MB), backward 29.2 (126 MB) and 5.5 for the weights' sums.
// (Weights and angles read one by one behind conditions, a row found by a division a lane:
// 34.6, 25.9 and 33.0.)
#include <math.h>

#include "rotary_common.h"

namespace {

constexpr int kNormThreads = 256;
constexpr int kNormMaxD = 256;

struct NormRows {  // one side's tensors, strides in elements (batch, row, head)
  const void *x, *w;
  const void *g;   // backward: the output's gradient
  void *out;       // y, or dx
  long long xb, xt, xh, gb, gt, gh, ob, ot, oh;
  int heads;
  uint32_t inv;    // for div_by: of this side's heads (forward, in q's: of both sides')
};

__device__ __forceinline__ float norm_load(const void *p, int dt, size_t i) {
  return dt == SF_F32 ? ((const float *)p)[i] : dt == SF_F16 ? (float)((const f16 *)p)[i] : sf_bf16_to_f32(((const uint16_t *)p)[i]);
}

// What a lane holds of a head: N pairs (a, b); b is absent (two() false) for dims that do
// not turn in the half layout and for dims past the rotated ones that have no partner.
//   VEC, half:        a = 16 bytes at d, b = 16 bytes at d + P (turned items only)
//   VEC, interleaved: the pairs of 16 bytes
//   else:             up to 4 pairs, or single dims past the rotated part, 64 lanes apart
template <int DT, bool VEC, bool INTER>
struct Held {
  static constexpr int E = Vec<DT>::E, N = !VEC ? 4 : INTER ? E / 2 : E;
  float a[N], b[N];

  struct At {
    int i, P, D, per, turned;  // item of its head, pairs, dims, items, those that turn
    bool live;                 // (lanes past a head's items hold zeros)
    __device__ __forceinline__ int d1(int j) const {
      if constexpr (!VEC) {
        const int e = i + 64 * j;
        return e < P ? (INTER ? 2 * e : e) : P + e;
      } else {
        const int d = i < turned ? i * E : (INTER ? 0 : P) + i * E;
        return d + (INTER ? 2 * j : j);
      }
    }
    __device__ __forceinline__ int d2(int j) const { return d1(j) + (INTER ? 1 : P); }
    __device__ __forceinline__ bool one(int j) const { return VEC ? live : live && i + 64 * j < per; }
    __device__ __forceinline__ bool two(int j) const {
      if constexpr (!VEC) return live && i + 64 * j < P;
      else return live && (INTER || i < turned);
    }
    __device__ __forceinline__ bool turns(int j) const { return VEC ? i < turned : i + 64 * j < P; }
    __device__ __forceinline__ int pair(int j) const { return VEC ? (INTER ? i * E / 2 : i * E) + j : i + 64 * j; }
  };

  // The weights of what the lane holds, and the cos and sin of its pairs, without branches: VEC,
  // neighbouring entries of LDS; where it holds nothing (zeros), or nothing that turns, the first ones.
  static __device__ __forceinline__ void weights(const float *w, const At &x, float (&wa)[N], float (&wb)[N]) {
    const int d = VEC && x.live ? x.d1(0) : 0, d2 = VEC && !INTER && x.live && x.i < x.turned ? d + x.P : d;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      wa[j] = w[!VEC ? (x.one(j) ? x.d1(j) : 0) : INTER ? d + 2 * j : d + j];
      wb[j] = w[!VEC ? (x.two(j) ? x.d2(j) : 0) : INTER ? d + 2 * j + 1 : d2 + j];
    }
  }
  static __device__ __forceinline__ void angles(const float2_t *c, const At &x, float2_t (&cs)[N]) {
    const int p = VEC && x.turns(0) ? x.pair(0) : 0;
#pragma unroll
    for (int j = 0; j < N; ++j) cs[j] = c[VEC ? p + j : x.turns(j) ? x.pair(j) : 0];
  }

  // the bits of a head, loaded before they are needed
  struct Bits {
    u32x4 lo, hi;
    float s1[VEC ? 1 : N], s2[VEC ? 1 : N];
  };
  static __device__ __forceinline__ Bits fetch(const void *p, size_t at, const At &x) {
    Bits v;
    constexpr int sz = DT == SF_F32 ? 4 : 2;
    if constexpr (VEC) {
      v.lo = v.hi = u32x4{0u, 0u, 0u, 0u};
      if (x.live) {
        const char *c = (const char *)p + (at + x.d1(0)) * sz;
        v.lo = *(const u32x4 *)c;
        if (!INTER && x.i < x.turned) v.hi = *(const u32x4 *)(c + x.P * sz);
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        v.s1[j] = x.one(j) ? sf_load_as_f32<DT>(p, at + x.d1(j)) : 0.f;
        v.s2[j] = x.two(j) ? sf_load_as_f32<DT>(p, at + x.d2(j)) : 0.f;
      }
    }
    return v;
  }
  __device__ __forceinline__ void set(const Bits &v) {
    if constexpr (!VEC) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        a[j] = v.s1[j];
        b[j] = v.s2[j];
      }
    } else {
      Vec<DT> p;
      p.load(v.lo);
      if constexpr (INTER) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          a[j] = p.v[2 * j];
          b[j] = p.v[2 * j + 1];
        }
      } else {
        Vec<DT> q;
        q.load(v.hi);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          a[j] = p.v[j];
          b[j] = q.v[j];
        }
      }
    }
  }
  __device__ __forceinline__ void store(void *p, size_t at, const At &x) const {
    constexpr int sz = DT == SF_F32 ? 4 : 2;
    if constexpr (!VEC) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (x.one(j)) sf_store_from_f32<DT>(p, at + x.d1(j), sf_opaque(a[j]));
        if (x.two(j)) sf_store_from_f32<DT>(p, at + x.d2(j), sf_opaque(b[j]));
      }
    } else if (x.live) {
      char *c = (char *)p + (at + x.d1(0)) * sz;
      Vec<DT> v;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if constexpr (INTER) {
          v.v[2 * j] = a[j];
          v.v[2 * j + 1] = b[j];
        } else {
          v.v[j] = a[j];
        }
      }
      *(u32x4 *)c = v.pack();
      if (!INTER && x.i < x.turned) {
#pragma unroll
        for (int j = 0; j < N; ++j) v.v[j] = b[j];
        *(u32x4 *)(c + x.P * sz) = v.pack();
      }
    }
  }
};

// The turned pair.
__device__ __forceinline__ float2_t norm_turn(float x1, float x2, float2_t cs) {
  return float2_t{fmaf(-x2, cs.y, x1 * cs.x), fmaf(x1, cs.y, x2 * cs.x)};
}

struct NormCut {
  int per, turned, lanes_log2, n_heads;  // items a head, those that turn, log2 of its lanes, heads of a launch (or side)
  uint32_t inv_T, inv_P;                 // for div_by
};

// The rows and heads of a workgroup's consecutive heads first ..: its first one's by (uniform)
// divisions, the others' by what they are past it.
struct NormAt {
  int row0, off0, b0, t0, heads, T;
  uint32_t inv_heads, inv_T;
  __device__ __forceinline__ NormAt(int first, int heads, int T, uint32_t inv_heads, uint32_t inv_T)
      : heads(heads), T(T), inv_heads(inv_heads), inv_T(inv_T) {
    row0 = first / heads;
    off0 = first - row0 * heads;
    b0 = row0 / T;
    t0 = row0 - b0 * T;
  }
  // the row past the first one, and the head, of the workgroup's head `past` (under 257; the
  // quotients' operands stay below 2^16, or the quotient is 0 or 1)
  __device__ __forceinline__ int row(int past, int &h) const {
    const int e = off0 + past, r = heads < 32768 ? div_by(e, inv_heads) : e >= heads;
    h = e - r * heads;
    return r;
  }
  __device__ __forceinline__ void token(int r, int &b, int &t) const {
    const int x = t0 + r, n = T < 32768 ? div_by(x, inv_T) : x >= T;
    b = b0 + n;
    t = x - n * T;
  }
};

// The lanes' table of cos and sin, one entry a (row, pair), of the workgroup's first `rows` rows.
__device__ __forceinline__ void norm_table(float2_t *cs, const NormAt &w, int rows, int P, uint32_t inv_P, RotaryPos pos,
                                           const double *inv_freq, float scale) {
  for (int i = threadIdx.x; i < rows * P; i += kNormThreads) {
    const int r = div_by(i, inv_P);
    int b, t;
    w.token(r, b, t);
    cs[i] = rotary_cs(pos.at(b, t), inv_freq[i - r * P], scale);
  }
}

// 256 / L heads a workgroup, one a group of L lanes: the loads fly while the table is made.
template <int DT, bool VEC, bool INTER>
__global__ void __launch_bounds__(kNormThreads)
k_qk_norm(NormRows q, NormRows k, int wdt, float eps, RotaryPos pos, const double *__restrict__ inv_freq, int P,
          float scale, int T, int D, NormCut cut) {
  using H = Held<DT, VEC, INTER>;
  constexpr int N = H::N;
  extern __shared__ __attribute__((aligned(16))) float smem[];
  float *const ws = smem;                              // [2][D] weights
  float2_t *const cs = (float2_t *)(smem + 2 * D);     // [rows][P]
  const int heads = q.heads + k.heads, hb = kNormThreads >> cut.lanes_log2, L = 1 << cut.lanes_log2;
  const int first = blockIdx.x * hb, slot = threadIdx.x >> cut.lanes_log2, count = min(hb, cut.n_heads - first);
  const NormAt w(first, heads, T, q.inv, cut.inv_T);
  int hh, b, t, unused;
  const int dr = w.row(min(slot, count - 1), hh), rows = w.row(count - 1, unused) + 1;
  w.token(dr, b, t);
  const bool is_q = hh < q.heads, live = slot < count;
  const int h = is_q ? hh : hh - q.heads, i = threadIdx.x & (L - 1);
  const typename H::At at = {i, P, D, cut.per, cut.turned, i < cut.per};
  H v;
  v.set(H::fetch(is_q ? q.x : k.x, (size_t)(is_q ? b * q.xb + t * q.xt + h * q.xh : b * k.xb + t * k.xt + h * k.xh), at));
  for (int d = threadIdx.x; d < 2 * D; d += kNormThreads) {
    if (d < D) ws[d] = norm_load(q.w, wdt, d);
    else if (k.heads) ws[d] = norm_load(k.w, wdt, d - D);
  }
  norm_table(cs, w, rows, P, cut.inv_P, pos, inv_freq, scale);
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) ss = fmaf(v.a[j], v.a[j], fmaf(v.b[j], v.b[j], ss));
  const float r = 1.f / sqrtf(sf_group_tree_sum(ss, L) / (float)D + eps);
  __syncthreads();
  float wa[N], wb[N];
  float2_t c[N];
  H::weights(ws + (is_q ? 0 : D), at, wa, wb);
  H::angles(cs + dr * P, at, c);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float y1 = v.a[j] * r * wa[j], y2 = v.b[j] * r * wb[j];
    const float2_t y = norm_turn(y1, y2, c[j]);
    v.a[j] = at.turns(j) ? y.x : y1;
    v.b[j] = at.turns(j) ? y.y : y2;
  }
  if (live) v.store(is_q ? q.out : k.out, (size_t)(is_q ? b * q.ob + t * q.ot + h * q.oh : b * k.ob + t * k.ot + h * k.oh), at);
}

// Backward. The first nq workgroups take q's heads, the others k's, each a run of `run`
// chunks of 256 / L heads; a lane sums its dims' g n over them, the workgroup's groups are
// then summed in LDS into one row of partials, which the second launch sums.
template <int DT, bool VEC, bool INTER>
__global__ void __launch_bounds__(kNormThreads)
k_qk_norm_back(NormRows q, NormRows k, int wdt, float eps, RotaryPos pos, const double *__restrict__ inv_freq, int P,
               float scale, int T, int D, NormCut cut, int n_rows, int nq, int run, float *__restrict__ part) {
  using H = Held<DT, VEC, INTER>;
  constexpr int N = H::N;
  extern __shared__ __attribute__((aligned(16))) float smem[];
  const bool is_q = (int)blockIdx.x < nq;
  const NormRows &x = is_q ? q : k;
  const int blk = is_q ? blockIdx.x : blockIdx.x - nq, heads = x.heads, n_heads = n_rows * heads;
  const int hb = kNormThreads >> cut.lanes_log2, L = 1 << cut.lanes_log2;
  const int slot = threadIdx.x >> cut.lanes_log2, i = threadIdx.x & (L - 1);
  float *const ws = smem;                      // [D]
  float2_t *const cs = (float2_t *)(smem + D + (D & 1));  // [rows][P]
  const typename H::At at = {i, P, D, cut.per, cut.turned, i < cut.per};
  for (int d = threadIdx.x; d < D; d += kNormThreads) ws[d] = norm_load(x.w, wdt, d);
  float da[N], db[N];
#pragma unroll
  for (int j = 0; j < N; ++j) da[j] = db[j] = 0.f;
  for (int u = 0; u < run; ++u) {
    const long long first_ = ((long long)blk * run + u) * hb;
    if (first_ >= n_heads) break;
    const int count = min(hb, n_heads - (int)first_);
    const NormAt w((int)first_, heads, T, x.inv, cut.inv_T);
    int h, b, t, unused;
    const int dr = w.row(min(slot, count - 1), h), rows = w.row(count - 1, unused) + 1;
    w.token(dr, b, t);
    const bool live = slot < count;
    const auto xb = H::fetch(x.x, (size_t)(b * x.xb + t * x.xt + h * x.xh), at);
    const auto gb = H::fetch(x.g, (size_t)(b * x.gb + t * x.gt + h * x.gh), at);
    __syncthreads();  // the last chunk's table is read
    norm_table(cs, w, rows, P, cut.inv_P, pos, inv_freq, scale);
    __syncthreads();
    H v, g;
    v.set(xb);
    g.set(gb);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) ss = fmaf(v.a[j], v.a[j], fmaf(v.b[j], v.b[j], ss));
    const float r = 1.f / sqrtf(sf_group_tree_sum(ss, L) / (float)D + eps);
    float wa[N], wb[N];
    float2_t c[N];
    H::weights(ws, at, wa, wb);
    H::angles(cs + dr * P, at, c);
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float2_t y = norm_turn(g.a[j], g.b[j], float2_t{c[j].x, -c[j].y});  // turned back: the opposite angle
      g.a[j] = at.turns(j) ? y.x : g.a[j];
      g.b[j] = at.turns(j) ? y.y : g.b[j];
      v.a[j] *= r;
      v.b[j] *= r;
      da[j] = live ? fmaf(g.a[j], v.a[j], da[j]) : da[j];
      db[j] = live ? fmaf(g.b[j], v.b[j], db[j]) : db[j];
      g.a[j] *= wa[j];
      g.b[j] *= wb[j];
      dot = fmaf(g.a[j], v.a[j], fmaf(g.b[j], v.b[j], dot));
    }
    dot = sf_group_tree_sum(dot, L) / (float)D;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      g.a[j] = r * fmaf(-v.a[j], dot, g.a[j]);
      g.b[j] = r * fmaf(-v.b[j], dot, g.b[j]);
    }
    if (live) g.store(x.out, (size_t)(b * x.ob + t * x.ot + h * x.oh), at);
  }
  __syncthreads();
  float *const sums = smem;  // [groups][D]
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (at.one(j)) sums[slot * D + at.d1(j)] = da[j];
    if (at.two(j)) sums[slot * D + at.d2(j)] = db[j];
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kNormThreads) {
    float s = 0.f;
    for (int n = 0; n < hb; ++n) s += sums[n * D + d];
    part[(size_t)blockIdx.x * D + d] = s;
  }
}

// The partials' sums, in a fixed order, rounded once to the weights' type: a workgroup takes 4 dims of one side, 64 lanes each.
__global__ void __launch_bounds__(256)
k_qk_norm_weights(const float *__restrict__ part, int nq, int nk, int D, int wdt, void *__restrict__ dwq,
                  void *__restrict__ dwk) {
  const int lane = threadIdx.x & 63, per = (D + 3) / 4, side = blockIdx.x / per;
  const int d = (blockIdx.x - side * per) * 4 + (threadIdx.x >> 6);
  const int n0 = side ? nq : 0, n1 = side ? nq + nk : nq;
  float s = 0.f;
  if (d < D)
    for (int n = n0 + lane; n < n1; n += 64) s += part[(size_t)n * D + d];
  s = sf_wave_sum(s);
  if (d < D && lane == 0) sf_store_dt(side ? dwk : dwq, wdt, d, s);
}

// How heads are cut into items and lanes; vec: 16 bytes at a time where every head of every
// tensor starts on 16 bytes and its parts are whole vectors.
bool norm_cut(int dtype, int rot_pairs, int interleaved, int T, int D, uintptr_t all, const long long *s, int n,
              NormCut *cut) {
  const int E = dtype == SF_F32 ? 4 : 8, rest = D - 2 * rot_pairs, turn_dims = interleaved ? 2 * rot_pairs : rot_pairs;
  bool vec = rest % E == 0 && turn_dims % E == 0 && (all & 15) == 0;
  for (int i = 0; i < n; ++i) vec = vec && s[i] % E == 0;
  cut->turned = vec ? turn_dims / E : rot_pairs;
  cut->per = vec ? (turn_dims + rest) / E : rot_pairs + rest;
  cut->inv_T = div_inv(T);
  cut->inv_P = div_inv(rot_pairs);
  cut->lanes_log2 = 0;
  while ((1 << cut->lanes_log2) < (vec ? cut->per : 64)) ++cut->lanes_log2;
  return vec;
}

int norm_check(const void *positions, const double *inv_freq, int rot_pairs, int dtype, int wdt, int B, int T, int H,
               int KVH, int D) {
  SF_REQUIRE(B >= 0 && T >= 0 && H > 0 && KVH >= 0 && D > 0, SF_EINVAL,
             "invalid head norm shape B=%d T=%d H=%d KVH=%d D=%d", B, T, H, KVH, D);
  SF_REQUIRE(D <= kNormMaxD, SF_EUNSUPPORTED, "head_dim=%d: at most %d", D, kNormMaxD);
  SF_REQUIRE(rot_pairs > 0 && 2LL * rot_pairs <= D, SF_EINVAL, "%d rotated pairs in a head of %d", rot_pairs, D);
  SF_REQUIRE(dtype >= SF_F32 && dtype <= SF_BF16 && wdt >= SF_F32 && wdt <= SF_BF16, SF_EINVAL, "bad dtype");
  SF_REQUIRE((long long)B * T * (H + (long long)KVH) <= 0x7fffffffLL - 65536, SF_EINVAL,
             "%d x %d rows of %d heads exceed the grid", B, T, H + KVH);
  SF_REQUIRE((long long)B * T == 0 || (positions && inv_freq), SF_EINVAL, "null pointer argument");
  return SF_OK;
}

// Rows of the table that `hb` consecutive heads touch at most.
int norm_rows(int hb, int heads) { return (hb + heads - 2) / heads + 1; }

}  // namespace

#define SF_NORM_DT(KERNEL)                                   \
  do {                                                       \
    if (dtype == SF_F32) SF_NORM_V(KERNEL, SF_F32);          \
    else if (dtype == SF_F16) SF_NORM_V(KERNEL, SF_F16);     \
    else SF_NORM_V(KERNEL, SF_BF16);                         \
  } while (0)
#define SF_NORM_V(KERNEL, DT)                                \
  do {                                                       \
    if (vec && interleaved) KERNEL(DT, true, true);          \
    else if (vec) KERNEL(DT, true, false);                   \
    else if (interleaved) KERNEL(DT, false, true);           \
    else KERNEL(DT, false, false);                           \
  } while (0)

extern "C" int sf_qk_norm_rotary(const void *q, void *q_out, const void *k, void *k_out, int dtype,
                                 const void *q_weight, const void *k_weight, int weight_dtype, float eps,
                                 const void *positions, int pos_i64, int pos_per_seq, const double *inv_freq,
                                 int rot_pairs, float scale, int interleaved, int B, int T, int H, int KVH, int D,
                                 const long long *strides, void *stream) {
  if (int rc = norm_check(positions, inv_freq, rot_pairs, dtype, weight_dtype, B, T, H, KVH, D)) return rc;
  if (B == 0 || T == 0) return SF_OK;
  SF_REQUIRE(q && q_out && q_weight && (KVH == 0 || (k && k_out && k_weight)), SF_EINVAL, "null pointer argument");
  const long long dq = (long long)H * D, dk = (long long)KVH * D;
  const long long whole[12] = {T * dq, dq, D, T * dq, dq, D, T * dk, dk, D, T * dk, dk, D};
  const long long *s = strides ? strides : whole;
  const NormRows rq = {q, q_weight, nullptr, q_out, s[0], s[1], s[2], 0, 0, 0, s[3], s[4], s[5], H,
                       div_inv(H + KVH)};
  const NormRows rk = {k, k_weight, nullptr, k_out, s[6], s[7], s[8], 0, 0, 0, s[9], s[10], s[11], KVH, 0};
  NormCut cut;
  const bool vec = norm_cut(dtype, rot_pairs, interleaved, T, D,
                            (uintptr_t)q | (uintptr_t)q_out | (KVH ? (uintptr_t)k | (uintptr_t)k_out : 0), s, KVH ? 12 : 6, &cut);
  cut.n_heads = B * T * (H + KVH);
  const int hb = kNormThreads >> cut.lanes_log2;
  const size_t lds = 2 * (size_t)D * 4 + (size_t)norm_rows(hb, H + KVH) * rot_pairs * 8;
  const RotaryPos pos = {positions, pos_i64, pos_per_seq ? T : 0};
  const unsigned grid = (unsigned)((cut.n_heads + hb - 1) / hb);
  hipStream_t st = (hipStream_t)stream;
#define SF_NORM_F(DT, V, I) \
  k_qk_norm<DT, V, I><<<grid, kNormThreads, lds, st>>>(rq, rk, weight_dtype, eps, pos, inv_freq, rot_pairs, scale, T, D, cut)
  SF_NORM_DT(SF_NORM_F);
#undef SF_NORM_F
  return sf_check_launch("sf_qk_norm_rotary");
}

namespace {

// Workgroups of each side and the chunks that each takes: at most 1024 (four a CU) and one more.
void norm_blocks(long long rows, int H, int KVH, int hb, int *nq, int *nk, int *run) {
  const long long cq = (rows * H + hb - 1) / hb, ck = (rows * KVH + hb - 1) / hb;
  *run = (int)((cq + ck + 1023) / 1024);
  if (*run < 1) *run = 1;
  *nq = (int)((cq + *run - 1) / *run);
  *nk = (int)((ck + *run - 1) / *run);
}

}  // namespace

extern "C" size_t sf_qk_norm_backward_workspace_bytes(int B, int T, int H, int KVH, int D) {
  if (B <= 0 || T <= 0 || H <= 0 || KVH < 0 || D <= 0 || (long long)B * T * (H + (long long)KVH) > 0x7fffffffLL - 65536) return 0;
  return (size_t)(1024 + 2) * D * sizeof(float);
}

extern "C" int sf_qk_norm_rotary_backward(const void *q, const void *q_grad, void *dq_out, const void *k,
                                          const void *k_grad, void *dk_out, int dtype, const void *q_weight,
                                          const void *k_weight, int weight_dtype, void *dq_weight, void *dk_weight,
                                          float eps, const void *positions, int pos_i64, int pos_per_seq,
                                          const double *inv_freq, int rot_pairs, float scale, int interleaved, int B,
                                          int T, int H, int KVH, int D, const long long *strides, void *workspace,
                                          size_t workspace_bytes, void *stream) {
  if (int rc = norm_check(positions, inv_freq, rot_pairs, dtype, weight_dtype, B, T, H, KVH, D)) return rc;
  SF_REQUIRE(B > 0 && T > 0, SF_EINVAL, "no rows");
  SF_REQUIRE(q && q_grad && dq_out && q_weight && dq_weight &&
                 (KVH == 0 || (k && k_grad && dk_out && k_weight && dk_weight)),
             SF_EINVAL, "null pointer argument");
  SF_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 &&
                 workspace_bytes >= sf_qk_norm_backward_workspace_bytes(B, T, H, KVH, D),
             SF_EINVAL, "head norm workspace too small or not 16-byte aligned");
  const long long wq = (long long)H * D, wk = (long long)KVH * D;
  const long long whole[18] = {T * wq, wq, D, T * wq, wq, D, T * wq, wq, D, T * wk, wk, D, T * wk, wk, D, T * wk, wk, D};
  const long long *s = strides ? strides : whole;
  const NormRows rq = {q, q_weight, q_grad, dq_out, s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], H,
                       div_inv(H)};
  const NormRows rk = {k, k_weight, k_grad, dk_out, s[9], s[10], s[11], s[12], s[13], s[14], s[15], s[16], s[17], KVH,
                       KVH ? div_inv(KVH) : 0};
  NormCut cut;
  const bool vec = norm_cut(dtype, rot_pairs, interleaved, T, D,
                            (uintptr_t)q | (uintptr_t)q_grad | (uintptr_t)dq_out |
                                (KVH ? (uintptr_t)k | (uintptr_t)k_grad | (uintptr_t)dk_out : 0),
                            s, KVH ? 18 : 9, &cut);
  const int hb = kNormThreads >> cut.lanes_log2, rows = B * T;
  int nq, nk, run;
  norm_blocks(rows, H, KVH, hb, &nq, &nk, &run);
  const int heads = KVH && KVH < H ? KVH : H;  // (the fewer heads a row, the more rows a chunk touches)
  const size_t tab = ((size_t)D + 1) * 4 + (size_t)norm_rows(hb, heads) * rot_pairs * 8, sums = (size_t)hb * D * 4;
  const size_t lds = tab > sums ? tab : sums;
  const RotaryPos pos = {positions, pos_i64, pos_per_seq ? T : 0};
  hipStream_t st = (hipStream_t)stream;
  float *part = (float *)workspace;
#define SF_NORM_B(DT, V, I)                                                                                          \
  k_qk_norm_back<DT, V, I><<<nq + nk, kNormThreads, lds, st>>>(rq, rk, weight_dtype, eps, pos, inv_freq, rot_pairs, \
                                                               scale, T, D, cut, rows, nq, run, part)
  SF_NORM_DT(SF_NORM_B);
#undef SF_NORM_B
  k_qk_norm_weights<<<(KVH ? 2 : 1) * ((D + 3) / 4), 256, 0, st>>>(part, nq, nk, D, weight_dtype, dq_weight, dk_weight);
  return sf_check_launch("sf_qk_norm_rotary_backward");
}
#undef SF_NORM_V
#undef SF_NORM_DT
