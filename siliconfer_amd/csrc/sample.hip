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
// Bins: the logits' axis is cut at the multiples of T kDelta, the same places for
// every part of a row whatever its maximum. A weight is held relative to its bin's
// upper edge, e = exp(-kDelta (j + 1 - x / (T kDelta))), as the integer e 2^36
// rounded: sums within a bin are exact in any order, so the counting atomics change
// no result, and a token's share is off by at most 2^-37 of itself. Bins are joined
// in 64-bit floats in a fixed order. Tokens 40 nats and more below the maximum (256
// bins) weigh nothing.
//
// k_sample_bins: a workgroup a chunk of 8192 logits, held in registers: the chunk's
// maximum, then its 256 bins' counts and weights in one 64-bit LDS atomic an element
// (count << 50 | weight), and the list of its best elements, whole bins up to
// kListCap of them.
// k_sample_pick: a workgroup a row joins the chunks' bins. Each filter's end and the
// draw lie in one bin that the bins' prefix sums name; its elements come from the
// chunks' lists where these hold the whole bin, from the row again where not, and are
// ordered by counting. A bin of more than kBinCap elements (dense ties, temperatures
// that squeeze the row into few bins) is searched by radix selection over the order
// bits instead: eight bits a pass over the row.
#include <math.h>

#include "sf_common.h"

namespace {

typedef unsigned long long u64;
constexpr int kSampThreads = 1024;
constexpr int kSampWaves = kSampThreads / 64;
constexpr int kPerThread = 8;
constexpr int kChunk = kSampThreads * kPerThread;
constexpr int kBins = 256;
constexpr double kDelta = 0.15625;  // nats a bin
constexpr int kListCap = 128;       // elements of a chunk's list
constexpr int kBinCap = 1024;       // elements of a bin ordered by counting
constexpr int kCountShift = 50;     // 8192 weights of up to 2^36 take 49 bits and a little
constexpr u64 kWeightMask = (1ull << kCountShift) - 1;

// Order-preserving bits of a logit (never 0); -inf and NaN share the lowest.
__device__ __forceinline__ uint32_t order_key(float x) {
  x = x != x ? -INFINITY : x;
  x = x == 0.f ? 0.f : x;
  const uint32_t u = sf_bitcast<uint32_t>(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return sf_bitcast<float>(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
constexpr uint32_t kNoKey = 0x007fffffu;  // order_key(-inf)

struct RowParams {
  float temperature, top_p, min_p;
  int top_k;
  const float *temperatures, *top_ps, *min_ps;
  const int *top_ks;
  __device__ __forceinline__ float t(int b) const { return temperatures ? temperatures[b] : temperature; }
};

// 1 / (T kDelta): a logit's place on the bins' axis is x times it. The floor keeps an
// infinite temperature from turning infinite logits into NaN.
__device__ __forceinline__ double bins_per_logit(float T) { return fmax(1.0 / ((double)T * kDelta), 1e-300); }

struct Binned {
  int bin;  // below the bin of `top`; kBins and more: no weight
  u64 w;
};
// Where x lies below the bin number `top` (a floor in 64 bits), and its weight. exp(-kDelta
// r) by its series about r = 1/2 to the seventh power: kDelta / 2 to the eighth over 8! is
// 3e-14. Explicit fmas, so that every kernel gets the same bits.
__device__ __forceinline__ Binned bin_of(float x, double per, double top) {
  const double t = (double)x * per, j = floor(t), below = j == top ? 0.0 : top - j;
  Binned r;
  r.bin = below < (double)kBins ? (int)below : kBins;  // (NaN: no weight)
  const double z = -kDelta * (j == t && isinf(t) ? -0.5 : (j - t) + 0.5);
  double p = 1.0 / 5040;
  p = fma(p, z, 1.0 / 720);
  p = fma(p, z, 1.0 / 120);
  p = fma(p, z, 1.0 / 24);
  p = fma(p, z, 1.0 / 6);
  p = fma(p, z, 0.5);
  p = fma(p, z, 1.0);
  p = fma(p, z, 1.0);
  // exp(-kDelta / 2) 2^36 p as an integer: the low bits of its sum with 2^52
  const double unit = 0.92484881321620482 * 68719476736.0;
  r.w = (u64)__double_as_longlong(fma(p, unit, 4503599627370496.0)) & ((1ull << 52) - 1);
  return r;
}

// What a chunk leaves in the workspace.
struct ChunkOut {
  double top;       // its maximum's bin number
  u64 best;         // its maximum: key << 32 | ~index
  int list_n, pad;
  u64 bins[kBins];  // count << kCountShift | weight
  u64 list[kListCap];
};

__device__ __forceinline__ u64 wave_max(u64 v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const u64 o = __shfl_xor(v, off, 64);
    v = o > v ? o : v;
  }
  return v;
}

template <int DT>
__global__ void __launch_bounds__(kSampThreads)
k_sample_bins(const void *__restrict__ logits, long long row_stride, int V, int chunks, RowParams rp,
              ChunkOut *__restrict__ outs) {
  __shared__ u64 bins[kBins];
  __shared__ u64 red[kSampWaves];
  __shared__ int list_bins, list_n;
  const int b = blockIdx.x / chunks, c = blockIdx.x - b * chunks;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const size_t row = (size_t)b * row_stride;
  ChunkOut *o = outs + blockIdx.x;
  const int i0 = c * kChunk + threadIdx.x;
  float x[kPerThread];
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const int i = i0 + k * kSampThreads;
    x[k] = i < V ? sf_load_as_f32<DT>(logits, row + i) : -INFINITY;
  }
  u64 best = 0;
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const u64 e = (u64)order_key(x[k]) << 32 | (uint32_t)~(i0 + k * kSampThreads);
    best = e > best ? e : best;
  }
  best = wave_max(best);
  if (lane == 0) red[wave] = best;
  if (threadIdx.x < kBins) bins[threadIdx.x] = 0;
  if (threadIdx.x == 0) list_n = 0;
  __syncthreads();
  best = red[0];
#pragma unroll
  for (int w = 1; w < kSampWaves; ++w) best = red[w] > best ? red[w] : best;
  const float T = rp.t(b), m = key_value((uint32_t)(best >> 32));
  const bool none = (uint32_t)(best >> 32) == kNoKey || !(T > 0.f);  // nothing here to weigh
  const double per = bins_per_logit(T), top = floor((double)m * per);
  if (threadIdx.x == 0) {
    o->top = top;
    o->best = best;
  }
  if (none) {
    if (threadIdx.x < kBins) o->bins[threadIdx.x] = 0;
    if (threadIdx.x == 0) o->list_n = 0;
    return;
  }
  int bin[kPerThread];
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const Binned e = bin_of(x[k], per, top);
    bin[k] = x[k] > -INFINITY ? e.bin : kBins;
    if (bin[k] < kBins) atomicAdd(&bins[bin[k]], 1ull << kCountShift | e.w);
  }
  __syncthreads();
  if (threadIdx.x < kBins) o->bins[threadIdx.x] = bins[threadIdx.x];
  if (wave == 0) {  // lane l: bins 4 l .. 4 l + 3; the list takes the bins that fit it
    int n[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) sum += n[j] = (int)(bins[4 * lane + j] >> kCountShift);
    int run = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(run, off, 64);
      if (lane >= off) run += v;
    }
    int before = run - sum, fit = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      before += n[j];
      fit += before <= kListCap;
    }
    const u64 whole = __ballot(fit == 4);
    const int full = whole == ~0ull ? 64 : __ffsll(~whole) - 1;  // lanes whose bins all fit
    fit = __shfl(fit, min(full, 63), 64);
    if (lane == 0) list_bins = full == 64 ? kBins : 4 * full + fit;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kPerThread; ++k)
    if (bin[k] < list_bins) {
      const int at = atomicAdd(&list_n, 1);
      o->list[at] = (u64)order_key(x[k]) << 32 | (uint32_t)~(i0 + k * kSampThreads);
    }
  __syncthreads();
  if (threadIdx.x == 0) o->list_n = list_n;
}

struct Found {   // a place in a bin's order: the r-th token (from 0) with this logit
  uint32_t key;
  u64 r;
  u64 upto;      // weight of the bin's tokens up to and with it
  int index;     // its index, where the search knows it, else -1
};

struct PickSmem {
  u64 w[kBins];       // the row's bins: integer weight
  int n[kBins];       // and count
  double before[kBins + 1], fac[kBins];  // weight before the bin, exp(-kDelta i) 2^-36
  int n_before[kBins + 1];
  u64 raw[kBinCap], el[kBinCap], run[kBinCap];
  u64 hist[256];
  u64 red[kSampWaves];
  u64 tmp[4];
  int n_raw, uncovered;
};

__device__ __forceinline__ u64 block_sum(u64 v, PickSmem &sm) {
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

template <int DT>
struct Row {
  const void *logits;
  size_t row;
  int V, chunks;
  double per, top;
  const ChunkOut *outs;
  PickSmem &sm;
  int held;  // the bin whose elements lie in sm.el, in order (-1: none)

  __device__ __forceinline__ float at(int i) const { return sf_load_as_f32<DT>(logits, row + i); }
  __device__ __forceinline__ u64 weight(uint32_t key) const { return bin_of(key_value(key), per, top).w; }
  __device__ __forceinline__ bool in(float x, int bin) const {
    return x > -INFINITY && bin_of(x, per, top).bin == bin;
  }

  // The elements of a bin of at most kBinCap into sm.el in order, running weights into sm.run.
  __device__ void hold(int bin) {
    if (held == bin) return;
    held = bin;
    const int n = sm.n[bin];
    __syncthreads();
    if (threadIdx.x == 0) sm.n_raw = sm.uncovered = 0;
    __syncthreads();
    // a chunk's list has the bin where its elements up to it fit the list
    for (int c = threadIdx.x >> 6; c < chunks; c += kSampWaves) {
      const ChunkOut &o = outs[c];
      const double shift = o.top == top ? 0.0 : top - o.top;
      const int ln = o.list_n, lane = threadIdx.x & 63;
      int here = 0, listed = 0;  // the chunk's elements in the bin, and of them in its list
      if (shift <= (double)bin) here = (int)(o.bins[bin - (int)shift] >> kCountShift);
      for (int i = lane; i - lane < ln; i += 64) {
        const u64 e = i < ln ? o.list[i] : 0;
        const bool is = i < ln && in(key_value((uint32_t)(e >> 32)), bin);
        if (is) sm.raw[atomicAdd(&sm.n_raw, 1)] = e;
        listed += __popcll(__ballot(is));
      }
      if (lane == 0 && listed < here) sm.uncovered = 1;
    }
    __syncthreads();
    if (sm.uncovered) {
      __syncthreads();
      if (threadIdx.x == 0) sm.n_raw = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < V; i += kSampThreads) {
        const float x = at(i);
        if (in(x, bin)) sm.raw[atomicAdd(&sm.n_raw, 1)] = (u64)order_key(x) << 32 | (uint32_t)~i;
      }
      __syncthreads();
    }
    if ((int)threadIdx.x < n) {
      const u64 e = sm.raw[threadIdx.x];
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += sm.raw[i] > e;
      sm.el[rank] = e;
    }
    __syncthreads();
    // running weights: a wave's scan, then the waves before it
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u64 run = (int)threadIdx.x < n ? weight((uint32_t)(sm.el[threadIdx.x] >> 32)) : 0;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const u64 v = __shfl_up(run, off, 64);
      if (lane >= off) run += v;
    }
    if (lane == 63) sm.red[wave] = run;
    __syncthreads();
    for (int w = 0; w < wave; ++w) run += sm.red[w];
    sm.run[threadIdx.x] = run;
    __syncthreads();
  }

  // The bin's first token whose running count, or weight, exceeds x (the last where none does).
  __device__ Found find(int bin, double x, bool by_count) {
    const int n = sm.n[bin];
    if (n <= kBinCap) {
      hold(bin);
      const int t = threadIdx.x;
      const bool over = t < n && (by_count ? (double)(t + 1) : (double)sm.run[t]) > x;
      const int passed = (int)block_sum(t < n && !over, sm);
      const int j = min(passed, n - 1);
      const uint32_t key = (uint32_t)(sm.el[j] >> 32);
      const u64 r = block_sum(t < j && (uint32_t)(sm.el[t] >> 32) == key, sm);
      return Found{key, r, sm.run[j], (int)~(uint32_t)sm.el[j]};
    }
    // radix selection over the order bits of the bin's elements
    const u64 all = by_count ? (u64)n : sm.w[bin];
    const u64 target = x >= (double)all ? all - 1 : x > 0 ? (u64)x : 0;
    uint32_t prefix = 0, mask = 0;
    u64 above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (threadIdx.x < 256) sm.hist[threadIdx.x] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < V; i += kSampThreads) {
        const float v = at(i);
        const uint32_t k = order_key(v);
        if ((k & mask) == prefix && v > -INFINITY) {
          const Binned e = bin_of(v, per, top);
          if (e.bin == bin) atomicAdd(&sm.hist[k >> shift & 255], by_count ? 1ull : e.w);
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
        if (before <= target && target < above + run) {
          int digit = -1;
          u64 start = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (digit < 0 && target < before + d[j]) {
              digit = 255 - 4 * threadIdx.x - j;
              start = before;
            }
            before += d[j];
          }
          sm.tmp[0] = digit;
          sm.tmp[1] = start;
        }
      }
      __syncthreads();
      prefix |= (uint32_t)sm.tmp[0] << shift;
      mask |= 255u << shift;
      above = sm.tmp[1];
    }
    const u64 w = weight(prefix), r = by_count ? target - above : (target - above) / w;
    u64 upto = above + (r + 1) * w;
    if (by_count) {  // the weight above it has not been summed yet
      u64 s = 0;
      for (int i = threadIdx.x; i < V; i += kSampThreads) {
        const float v = at(i);
        if (order_key(v) > prefix && in(v, bin)) s += bin_of(v, per, top).w;
      }
      upto = block_sum(s, sm) + (r + 1) * w;
    }
    return Found{prefix, r, upto, -1};
  }

  // Tokens of the bin with this logit.
  __device__ u64 ties(int bin, uint32_t key) {
    u64 c = 0;
    if (sm.n[bin] <= kBinCap) {
      hold(bin);
      c = (int)threadIdx.x < sm.n[bin] && (uint32_t)(sm.el[threadIdx.x] >> 32) == key;
    } else {
      for (int i = threadIdx.x; i < V; i += kSampThreads) c += order_key(at(i)) == key;
    }
    return block_sum(c, sm);
  }

  // Count and weight of the bin's tokens that weigh at least `least` of the largest.
  __device__ void heavy(int bin, double M, double inv_t, uint32_t kmax, double least, u64 *count, u64 *sum) {
    auto is = [&](uint32_t k) {
      return k == kmax || exp(((double)key_value(k) - M) * inv_t) >= least;
    };
    u64 c = 0, s = 0;
    if (sm.n[bin] <= kBinCap) {
      hold(bin);
      if ((int)threadIdx.x < sm.n[bin]) {
        const uint32_t k = (uint32_t)(sm.el[threadIdx.x] >> 32);
        c = is(k);
        s = c ? weight(k) : 0;
      }
    } else {
      for (int i = threadIdx.x; i < V; i += kSampThreads) {
        const float v = at(i);
        if (in(v, bin) && is(order_key(v))) {
          ++c;
          s += bin_of(v, per, top).w;
        }
      }
    }
    *count = block_sum(c, sm);
    *sum = block_sum(s, sm);
  }

  // The index of the r-th token with this logit.
  __device__ int index_of(uint32_t key, u64 r) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int per_wave = ((V + kSampWaves - 1) / kSampWaves + 63) & ~63;
    const int lo = min(wave * per_wave, V), hi = min(lo + per_wave, V);
    u64 n = 0;
    for (int i = lo; i < hi; i += 64) n += __popcll(__ballot(i + lane < hi && order_key(at(min(i + lane, V - 1))) == key));
    __syncthreads();
    if (lane == 0) sm.red[wave] = n;
    __syncthreads();
    u64 before = 0;
    for (int w = 0; w < wave; ++w) before += sm.red[w];
    if (before <= r && r < before + n)
      for (int i = lo; i < hi; i += 64) {
        const u64 m = __ballot(i + lane < hi && order_key(at(min(i + lane, V - 1))) == key);
        if ((m >> lane & 1) && before + __popcll(m & ((1ull << lane) - 1)) == r) sm.tmp[2] = i + lane;
        before += __popcll(m);
      }
    __syncthreads();
    return (int)sm.tmp[2];
  }

  // The first bin up to `last` whose weight, with that of the bins before it, exceeds x.
  __device__ int bin_past(double x, int last) {
    const int t = threadIdx.x;
    const int j = (int)block_sum(t <= last && t < kBins && !(sm.before[t + 1] > x), sm);
    return min(j, last);
  }
};

template <int DT>
__global__ void __launch_bounds__(kSampThreads)
k_sample_pick(const void *__restrict__ logits, long long row_stride, int V, int chunks, const float *__restrict__ u,
              RowParams rp, const ChunkOut *__restrict__ outs, int32_t *__restrict__ tokens,
              float *__restrict__ logprobs) {
  __shared__ PickSmem sm;
  const int b = blockIdx.x, lane = threadIdx.x & 63;
  const ChunkOut *o = outs + (size_t)b * chunks;
  u64 best = 0;
  for (int c = lane; c < chunks; c += 64) best = o[c].best > best ? o[c].best : best;
  best = wave_max(best);
  const uint32_t kmax = (uint32_t)(best >> 32);
  const float T = rp.t(b);
  const bool empty = kmax == kNoKey;
  if (empty || !(T > 0.f)) {
    if (threadIdx.x == 0) {
      tokens[b] = empty ? -1 : (int)~(uint32_t)best;
      if (logprobs) logprobs[b] = empty ? -INFINITY : 0.f;
    }
    return;
  }
  const double M = (double)key_value(kmax), inv_t = fmax(1.0 / (double)T, 1e-300), per = bins_per_logit(T);
  Row<DT> row = {logits, (size_t)b * row_stride, V, chunks, per, floor(M * per), o, sm, -1};
  // the row's bins: four threads a bin, each every fourth chunk
  {
    const int bin = threadIdx.x & (kBins - 1), part = threadIdx.x / kBins;
    u64 n = 0, w = 0;
    for (int c = part; c < chunks; c += kSampThreads / kBins) {
      const double shift = o[c].top == row.top ? 0.0 : row.top - o[c].top;
      if (shift <= (double)bin) {
        const u64 v = o[c].bins[bin - (int)shift];
        n += v >> kCountShift;
        w += v & kWeightMask;
      }
    }
    sm.raw[threadIdx.x] = n;
    sm.el[threadIdx.x] = w;
    __syncthreads();
    if (threadIdx.x < kBins) {
#pragma unroll
      for (int j = 1; j < kSampThreads / kBins; ++j) {
        n += sm.raw[threadIdx.x + j * kBins];
        w += sm.el[threadIdx.x + j * kBins];
      }
      sm.n[bin] = (int)n;
      sm.w[bin] = w;
      sm.fac[bin] = exp(-kDelta * bin) * (1.0 / 68719476736.0);
    }
  }
  __syncthreads();
  if (threadIdx.x < 64) {  // prefix sums, lane l: bins 4 l .. 4 l + 3
    double v[4], sum = 0;
    int n[4], ns = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sum += v[j] = (double)sm.w[4 * lane + j] * sm.fac[4 * lane + j];
      ns += n[j] = sm.n[4 * lane + j];
    }
    double run = sum;
    int nrun = ns;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double a = __shfl_up(run, off, 64);
      const int d = __shfl_up(nrun, off, 64);
      if (lane >= off) {
        run += a;
        nrun += d;
      }
    }
    double at = __shfl_up(run, 1, 64);  // the sum before the lane's bins
    if (lane == 0) at = 0;
    int nat = nrun - ns;
    if (lane == 0) sm.before[0] = 0, sm.n_before[0] = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      at += v[j];
      nat += n[j];
      sm.before[4 * lane + j + 1] = j == 3 ? run : at;
      sm.n_before[4 * lane + j + 1] = nat;
    }
  }
  __syncthreads();
  // What stays: the bins before `last`, and of that bin the tokens before and with the
  // (r + 1)-th that has the logit `key`: `upto` of weight. At first everything.
  int last = kBins - 1;
  uint32_t key = 0;
  u64 r = ~0ull >> 1, upto = sm.w[kBins - 1];
  auto weight_kept = [&]() { return sm.before[last] + (double)upto * sm.fac[last]; };
  const int k = rp.top_ks ? rp.top_ks[b] : rp.top_k;
  if (k > 0 && k < sm.n_before[kBins]) {
    const int t = threadIdx.x;
    last = (int)block_sum(t < kBins && sm.n_before[t + 1] < k, sm);
    const Found f = row.find(last, (double)(k - 1 - sm.n_before[last]), true);
    const u64 n = row.ties(last, f.key);
    key = f.key;
    upto = f.upto + (n - 1 - f.r) * row.weight(key);
    r = n - 1;
  }
  const float tp = rp.top_ps ? rp.top_ps[b] : rp.top_p;
  if (tp < 1.f) {
    const double bound = fmax((double)tp, 0.0) * weight_kept();
    const int bin = row.bin_past(bound, last);
    const Found f = row.find(bin, (bound - sm.before[bin]) / sm.fac[bin], false);
    if (bin < last || f.key > key || (f.key == key && f.r < r)) {
      last = bin;
      key = f.key;
      r = f.r;
      upto = f.upto;
    }
  }
  const float mp = rp.min_ps ? rp.min_ps[b] : rp.min_p;
  if (mp > 0.f) {
    const double least = fmin((double)mp, 1.0), below = row.top - floor(M * per + log(least) * (1.0 / kDelta));
    const int bin = below < (double)kBins ? max(0, (int)below) : kBins;  // (an infinite M: bin 0 by the next line)
    const int at = isinf(M) ? 0 : bin;
    if (at <= last) {
      u64 n, w;
      row.heavy(at, M, inv_t, kmax, least, &n, &w);
      if (at < last || w < upto) {
        last = at;
        upto = w;
        key = 0;  // which of them: those that weigh enough, all before any other
        r = ~0ull >> 1;
      }
    }
  }
  const double total = weight_kept(), target = fmin(fmax((double)u[b], 0.0), 1.0) * total;
  int bin = row.bin_past(target, last);
  // (rounding, or a last bin of which nothing stays: the last token that does)
  while (bin > 0 && (bin == last ? upto == 0 : sm.w[bin] == 0)) --bin;
  double x = (target - sm.before[bin]) / sm.fac[bin];
  const double most = (double)(bin == last ? upto : sm.w[bin]);
  if (!(x < most)) x = most - 1.0;
  const Found f = row.find(bin, x, false);
  const int token = f.index >= 0 ? f.index : row.index_of(f.key, f.r);
  if (threadIdx.x == 0) {
    tokens[b] = token;
    if (logprobs)
      logprobs[b] = (float)((f.key == kmax ? 0.0 : ((double)key_value(f.key) - M) * inv_t) -
                            log(total / ((double)row.weight(kmax) * sm.fac[0])));
  }
}

}  // namespace

static long long sample_chunks(int V) { return ((long long)V + kChunk - 1) / kChunk; }

extern "C" size_t sf_sample_workspace_bytes(int B, int V) {
  if (B <= 0 || V <= 0) return 0;
  return (size_t)B * sample_chunks(V) * sizeof(ChunkOut);
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
  const long long chunks = sample_chunks(V);
  SF_REQUIRE(B * chunks <= 0x7fffffffLL, SF_EINVAL, "B=%d rows of %d exceed the grid", B, V);
  SF_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0, SF_EINVAL, "workspace must be 256-byte aligned");
  const size_t need = sf_sample_workspace_bytes(B, V);
  SF_REQUIRE(workspace_bytes >= need, SF_EINVAL, "sampling workspace too small: %zu < %zu", workspace_bytes, need);
  const RowParams rp = {temperature, top_p, min_p, top_k, temperatures, top_ps, min_ps, top_ks};
  ChunkOut *outs = (ChunkOut *)workspace;
  hipStream_t st = (hipStream_t)stream;
#define SF_SAMP(DT)                                                                                                \
  do {                                                                                                             \
    k_sample_bins<DT><<<(unsigned)(B * chunks), kSampThreads, 0, st>>>(logits, row_stride, V, (int)chunks, rp, outs); \
    k_sample_pick<DT><<<B, kSampThreads, 0, st>>>(logits, row_stride, V, (int)chunks, u, rp, outs, tokens, logprobs); \
  } while (0)
  if (dtype == SF_F32) SF_SAMP(SF_F32);
  else if (dtype == SF_F16) SF_SAMP(SF_F16);
  else SF_SAMP(SF_BF16);
#undef SF_SAMP
  return sf_check_launch("sf_sample");
}
