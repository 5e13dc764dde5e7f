// sample.hip — a token a row from given random numbers (gfx950).
//
// A row's tokens are taken in descending order of their logits, equal logits by
// ascending index; NaN counts as -inf. With M the largest logit, token i weighs
// w_i = exp((x_i - M) / T). Of them stay, one filter after the other,
//   top-k   the k first and every token whose logit equals the k-th's,
//   top-p   those before which at most top_p of the weight left by top-k lies,
//   min-p   those with w_i >= min_p,
// each a prefix of the order. The token is the first whose running weight exceeds
// u times the weight that stays; T <= 0 takes the first token of the order. A row
// with no logit above -inf gives token -1 (log probability -inf); a logit of +inf
// weighs 1 and every finite one beside it 0.
//
// Weights come from 64-bit exponentials and are held as integers, w 2^S rounded,
// S = 62 - ceil(log2 V): sums of them are exact in 64 bits whatever their order, so
// the counting atomics below change no result, and a running weight is off by at
// most V 2^-(S+1) (2^-28 of the largest weight at V = 2^17).
//
// A place in the order ("the k-th token", "where the running weight passes x") is
// found by radix selection over the logits' order-preserving bits: eight bits a
// pass, each pass one read of the row and a histogram of counts or weights in LDS.
#include <math.h>

#include "sf_common.h"

namespace {

constexpr int kSampThreads = 1024;
constexpr int kSampWaves = kSampThreads / 64;
typedef unsigned long long u64;

__device__ __forceinline__ uint32_t order_key(float x) {
  x = x != x ? -INFINITY : x;
  x = x == 0.f ? 0.f : x;
  const uint32_t u = sf_bitcast<uint32_t>(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return sf_bitcast<float>(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct RowParams {
  float temperature, top_p, min_p;
  int top_k;
};

struct Weigh {  // a logit's weight from its order bits
  double M, inv_t, unit;  // unit = 2^S
  uint32_t kmax;
  __device__ __forceinline__ double real(uint32_t k) const {
    const float x = key_value(k);  // (-inf first: it weighs 0 at any temperature)
    return k == kmax ? 1.0 : x == -INFINITY ? 0.0 : exp(((double)x - M) * inv_t);
  }
  __device__ __forceinline__ u64 of(uint32_t k) const { return (u64)(real(k) * unit + 0.5); }
};

struct Place {   // a place in the order
  uint32_t key;  // the logit there
  u64 above;     // the count, or weight, of the tokens with larger logits
};

struct Smem {
  u64 hist[256];
  u64 red[kSampWaves];
  u64 found[2];
};

__device__ __forceinline__ u64 block_sum(u64 v, Smem &sm) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sm.red[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 s = 0;
#pragma unroll
  for (int w = 0; w < kSampWaves; ++w) s += sm.red[w];
  return s;
}

// The first place where the running sum of `mass` (of a token's key) over the order
// exceeds `target`; the caller has checked that the whole sum does.
template <class Key, class Mass>
__device__ Place locate(int V, u64 target, Key key, Mass mass, Smem &sm) {
  uint32_t prefix = 0, mask = 0;
  u64 above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) sm.hist[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += kSampThreads) {
      const uint32_t k = key(i);
      if ((k & mask) == prefix) {
        const u64 m = mass(k);
        if (m) atomicAdd(&sm.hist[k >> shift & 255], m);
      }
    }
    __syncthreads();
    if (threadIdx.x < 64) {  // lane l: digits 255 - 4 l down to 252 - 4 l
      u64 own = 0, d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) own += d[j] = sm.hist[255 - 4 * (int)threadIdx.x - j];
      u64 run = own;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const u64 o = __shfl_up(run, off, 64);
        if ((int)threadIdx.x >= off) run += o;
      }
      u64 before = above + run - own;
      if (before <= target && target < above + run)
        for (int j = 0; j < 4; ++j) {
          if (target < before + d[j]) {
            sm.found[0] = 255 - 4 * threadIdx.x - j;
            sm.found[1] = before;
            break;
          }
          before += d[j];
        }
    }
    __syncthreads();
    prefix |= (uint32_t)sm.found[0] << shift;
    mask |= 255u << shift;
    above = sm.found[1];
  }
  return Place{prefix, above};
}

template <int DT>
__global__ void __launch_bounds__(kSampThreads)
k_sample(const void *__restrict__ logits, long long row_stride, int V, const float *__restrict__ u,
         RowParams all, const float *__restrict__ temperatures, const int *__restrict__ top_ks,
         const float *__restrict__ top_ps, const float *__restrict__ min_ps, int scale_bits,
         int32_t *__restrict__ tokens, float *__restrict__ logprobs) {
  __shared__ Smem sm;
  __shared__ u64 tie_cnt[kSampWaves];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const size_t row = (size_t)b * row_stride;
  auto key = [&](int i) { return order_key(sf_load_as_f32<DT>(logits, row + i)); };
  RowParams p = all;
  if (temperatures) p.temperature = temperatures[b];
  if (top_ks) p.top_k = top_ks[b];
  if (top_ps) p.top_p = top_ps[b];
  if (min_ps) p.min_p = min_ps[b];
  // the largest logit, its lowest index: the largest of (key, ~index)
  u64 best = 0;
  for (int i = threadIdx.x; i < V; i += kSampThreads) {
    const u64 c = (u64)key(i) << 32 | (uint32_t)~i;
    best = c > best ? c : best;
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const u64 o = __shfl_xor(best, off, 64);
    best = o > best ? o : best;
  }
  if (lane == 0) sm.red[wave] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSampWaves; ++w) best = sm.red[w] > best ? sm.red[w] : best;
  const uint32_t kmax = (uint32_t)(best >> 32);
  const bool empty = kmax == order_key(-INFINITY);
  if (empty || !(p.temperature > 0.f)) {
    if (threadIdx.x == 0) {
      tokens[b] = empty ? -1 : (int)~(uint32_t)best;
      if (logprobs) logprobs[b] = empty ? -INFINITY : 0.f;
    }
    return;
  }
  const Weigh wt = {(double)key_value(kmax), fmax(1.0 / (double)p.temperature, 1e-300), (double)(1ull << scale_bits), kmax};
  // top-k: the k-th logit, the last that stays
  uint32_t k_last = 0;
  if (p.top_k > 0 && p.top_k < V)
    k_last = locate(V, (u64)p.top_k - 1, key, [](uint32_t) -> u64 { return 1; }, sm).key;
  auto mass = [&](uint32_t k) -> u64 { return k >= k_last ? wt.of(k) : 0; };
  u64 sum = 0;
  for (int i = threadIdx.x; i < V; i += kSampThreads) sum += mass(key(i));
  u64 total = block_sum(sum, sm);
  // top-p: up to the first token whose running weight exceeds top_p of the total
  uint32_t p_last = 0;
  if (p.top_p < 1.f) {
    const u64 bound = (u64)(fmax((double)p.top_p, 0.0) * (double)total);
    if (bound < total) {
      const Place at = locate(V, bound, key, mass, sm);
      const u64 w = wt.of(at.key);
      p_last = at.key;
      total = at.above + ((bound - at.above) / w + 1) * w;
    }
  }
  // min-p
  const double floor_w = fmin((double)p.min_p, 1.0);
  if (p.min_p > 0.f && !(wt.real(p_last > k_last ? p_last : k_last) >= floor_w)) {
    sum = 0;
    for (int i = threadIdx.x; i < V; i += kSampThreads) {
      const uint32_t k = key(i);
      sum += k >= k_last && k > p_last && wt.real(k) >= floor_w ? wt.of(k) : 0;
    }
    total = block_sum(sum, sm);
  }
  const double x = (double)u[b] * (double)total;
  u64 target = !(x > 0.0) ? 0 : x < (double)total ? (u64)x : total - 1;
  if (target >= total) target = total - 1;
  const Place at = locate(V, target, key, mass, sm);
  // its index: the r-th of the tokens with that logit
  const u64 w = wt.of(at.key), r = (target - at.above) / w;
  const int per = ((V + kSampWaves - 1) / kSampWaves + 63) & ~63;
  const int lo = min(wave * per, V), hi = min(lo + per, V);
  u64 ties = 0;
  for (int i0 = lo; i0 < hi; i0 += 64) ties += __popcll(__ballot(i0 + lane < hi && key(min(i0 + lane, V - 1)) == at.key));
  __syncthreads();
  if (lane == 0) tie_cnt[wave] = ties;
  __syncthreads();
  u64 before = 0;
  for (int v = 0; v < wave; ++v) before += tie_cnt[v];
  if (before <= r && r < before + ties)
    for (int i0 = lo; i0 < hi; i0 += 64) {
      const u64 m = __ballot(i0 + lane < hi && key(min(i0 + lane, V - 1)) == at.key);
      if ((m >> lane & 1) && before + __popcll(m & ((1ull << lane) - 1)) == r) {
        tokens[b] = i0 + lane;
        if (logprobs)
          logprobs[b] = (float)(log(wt.real(at.key)) - log((double)total / wt.unit));
      }
      before += __popcll(m);
    }
}

}  // namespace

extern "C" size_t sf_sample_workspace_bytes(int B, int V) {
  (void)B;
  (void)V;
  return 0;
}

extern "C" int sf_sample(const void *logits, int dtype, long long row_stride, int B, int V, const float *u,
                         float temperature, int top_k, float top_p, float min_p, const float *temperatures,
                         const int32_t *top_ks, const float *top_ps, const float *min_ps, int32_t *tokens,
                         float *logprobs, void *workspace, size_t workspace_bytes, void *stream) {
  SF_REQUIRE(B >= 0 && V > 0, SF_EINVAL, "invalid sampling shape B=%d V=%d", B, V);
  SF_REQUIRE(V <= (1 << 24), SF_EUNSUPPORTED, "V=%d: at most 16777216 tokens", V);
  SF_REQUIRE(dtype >= SF_F32 && dtype <= SF_BF16, SF_EINVAL, "bad dtype %d", dtype);
  SF_REQUIRE(row_stride >= 0, SF_EINVAL, "row stride %lld", row_stride);
  SF_REQUIRE(temperature == temperature && top_k >= 0 && top_p > 0.f && min_p >= 0.f && min_p <= 1.f, SF_EINVAL,
             "need top_k >= 0, top_p > 0, 0 <= min_p <= 1 (got %d, %g, %g; temperature %g)", top_k, top_p, min_p,
             temperature);
  if (B == 0) return SF_OK;
  SF_REQUIRE(logits && u && tokens, SF_EINVAL, "null pointer argument");
  (void)workspace;
  (void)workspace_bytes;
  int bits = 62;
  while ((1ll << (62 - bits)) < V) --bits;
  const RowParams all = {temperature, top_p, min_p, top_k};
  hipStream_t st = (hipStream_t)stream;
#define SF_SAMP(DT)                                                                                          \
  k_sample<DT><<<B, kSampThreads, 0, st>>>(logits, row_stride, V, u, all, temperatures, top_ks, top_ps, min_ps, \
                                           bits, tokens, logprobs)
  if (dtype == SF_F32) SF_SAMP(SF_F32);
  else if (dtype == SF_F16) SF_SAMP(SF_F16);
  else SF_SAMP(SF_BF16);
#undef SF_SAMP
  return sf_check_launch("sf_sample");
}
