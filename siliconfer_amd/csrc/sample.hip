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
// Bins: the logits' axis is cut at the multiples of T kDelta, the same places for every
// part of a row whatever its maximum. A weight is held relative to its bin's middle, as
// the integer 2^36 e^y, y within kDelta / 2: sums within a bin are exact in any order, so
// the counting atomics change no result, and a token's share is off by some 3e-10 of
// itself. Bins are joined in 64-bit floats in a fixed order. Tokens 32 nats and more below
// the maximum (256 bins, 1e-14 of its weight) weigh nothing.
//
// k_sample_bins: a workgroup a chunk of 10240 logits, held in registers: the chunk's
// maximum, then its 256 bins' counts and weights in one 64-bit LDS atomic an element
// (count << 50 | weight), and the list of its best elements, whole bins up to
// kListCap of them.
// k_sample_pick: a workgroup a row joins the chunks' bins. Where the bins up to the end of
// what the filters leave (or, without any, up to the draw) hold at most kHeadCap elements,
// these are gathered from the chunks' lists (from the row again where a list ends before
// them) and one wave orders them by counting and applies every rule to the ordered
// weights. Otherwise each filter's end and the draw are looked up one after the other in
// the one bin that the bins' prefix sums name; a bin of more than kBinCap elements (a large
// vocabulary's bulk, dense ties) is cut into 256 ranges of keys, a pass over the row, until
// the one that the search falls into can be ordered, as a rule after one pass.
// Measured (us, first + second launch; a workgroup a row with radix passes over it in
// brackets): 1 x 151936 fp32, top-k 50 and top-p, 6.6 + 8.8 (865); 64 x 151936 bf16, a
// row's own settings, 18.4 + 12.9 (993), of them 3.8 for the bytes at a copy's rate; at
// temperature alone a draw past the head re-reads its row: 8 x 32000 6.5 + 17.6 (6.8 with
// all draws within the head), of normal logits, none within it, 38 a call, 8 x 151936 114
// (the one workgroup's VALU: some 45 a pass). The first launch is bound by VALU issue (43
// instructions an element, two thirds of the time) and the five barriers of its
// workgroups, two a CU at a time; the second by the latency of some twenty dependent steps
// of one workgroup a row.
#include <math.h>

#include "sample_place.h"
#include "sf_common.h"

namespace {

typedef unsigned long long u64;
constexpr int kSampThreads = 1024;
constexpr int kSampWaves = kSampThreads / 64;
constexpr int kBinThreads = 1024;   // of the first kernel
constexpr int kBinWaves = kBinThreads / 64;
// Logits a thread holds. us a call in a replayed graph, fp32, top-k 50 and top-p, with 10 (4; 6; 8;
// 12): 1 x 32000 14.2 (13.7; 13.8; 14.1; 14.5), 64 x 32000 16.6 (17.1; 17.6; 16.6; 16.7), 64 x 50257
// 19.6 (22.4; 20.7; 19.1; 20.1), 1 x 151936 15.4 (18.6; 16.7; 16.0; 15.7), 64 x 151936 29.3 (41.1;
// 34.5; 31.2; 29.6).
constexpr int kPerThread = 10;
constexpr int kChunk = kBinThreads * kPerThread;
constexpr int kListCap = 128;       // elements of a chunk's list
constexpr int kBinCap = 1024;       // elements of a bin, or of a range of keys, ordered at once
constexpr int kHeadCap = 512;       // elements of the head: eight a lane of one wave
constexpr int kCountShift = 50;     // 10240 weights of up to 1.07 2^36 take 49.5 bits
constexpr u64 kWeightMask = (1ull << kCountShift) - 1;
static_assert(kChunk * 1.07 < (1ull << (kCountShift - 36)) && kChunk < (1 << (64 - kCountShift)), "a bin's weight and count");

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
  const int32_t *at;  // or null: row b's number is u[*at + at_add + b] of u_n, its token also hist[..]
  int32_t *hist;
  int at_add, u_n, B;
  __device__ __forceinline__ float t(int b) const { return temperatures ? temperatures[b] : temperature; }
  // where row b's number lies (kept inside u)
  __device__ __forceinline__ int place(int b) const {
    return at ? (int)max(0ll, min((long long)*at + at_add, (long long)u_n - B)) + b : b;
  }
};

// A row with infinite logits draws among them alone: they count as 0, all others as -inf.
__device__ __forceinline__ float flat_value(float x) { return x == INFINITY ? 0.f : -INFINITY; }

// What a chunk leaves in the workspace.
struct ChunkOut {
  double top;       // its maximum's bin number (inf: infinite logits)
  u64 best;         // its maximum: key << 32 | ~index
  int list_n, list_bins;  // the list's elements, the bins it has whole
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
__global__ void __launch_bounds__(kBinThreads)
k_sample_bins(const void *__restrict__ logits, long long row_stride, int V, int chunks, RowParams rp,
              ChunkOut *__restrict__ outs) {
  __shared__ u64 bins[kBins];
  __shared__ float red[kBinWaves];
  __shared__ uint2 list[kListCap];
  __shared__ int list_bins, list_n;
  const int b = blockIdx.x / chunks, c = blockIdx.x - b * chunks;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const size_t row = (size_t)b * row_stride;
  ChunkOut *o = outs + blockIdx.x;
  const int i0 = c * kChunk + threadIdx.x;
  float x[kPerThread];
  if ((c + 1) * kChunk <= V) {
    const size_t first = row + i0;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) x[k] = sf_load_as_f32<DT>(logits, first + k * kBinThreads);
  } else {
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int i = i0 + k * kBinThreads;
      x[k] = i < V ? sf_load_as_f32<DT>(logits, row + i) : -INFINITY;
    }
  }
  const float T = rp.t(b);
  float m = x[0];
#pragma unroll
  for (int k = 1; k < kPerThread; ++k) m = fmaxf(m, x[k]);  // (drops NaN; of NaN alone it is undone below)
  m = sf_wave_max(m != m ? -INFINITY : m);
  if (lane == 0) red[wave] = m;
  if (threadIdx.x < kBins) bins[threadIdx.x] = 0;
  if (threadIdx.x == 0) list_n = 0;
  __syncthreads();
  m = red[lane & (kBinWaves - 1)];
  m = sf_wave_max(m);
  if (!(T > 0.f)) {  // the largest logit's lowest index is all that counts
    u64 best = 0;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k)
      if (x[k] == m) {
        const u64 e = (u64)order_key(m) << 32 | (uint32_t)~(i0 + k * kBinThreads);
        best = e > best ? e : best;
      }
    best = wave_max(best);
    if (lane == 0) bins[wave] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kBinWaves; ++w) best = bins[w] > best ? bins[w] : best;
      o->best = best ? best : (u64)kNoKey << 32;
    }
    return;
  }
  if (threadIdx.x == 0) o->best = (u64)order_key(m) << 32;
  const bool flat = m == INFINITY;
  if (flat) {
    m = 0.f;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) x[k] = flat_value(x[k]);
  }
  const double per = bins_per_logit(T), top = m > -INFINITY ? top_bin(m, per) : -INFINITY;
  if (threadIdx.x == 0) o->top = flat ? INFINITY : top;
  if (!(m > -INFINITY)) {  // nothing here to weigh
    if (threadIdx.x < kBins) o->bins[threadIdx.x] = 0;
    if (threadIdx.x == 0) o->list_n = 0, o->list_bins = kBins;
    return;
  }
  int bin[kPerThread];
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const Binned e = bin_of(x[k], per, top, 1ull << kCountShift);
    bin[k] = e.bin;  // (-inf and NaN lie past the bins)
    if ((unsigned)bin[k] < (unsigned)kBins) atomicAdd(&bins[bin[k]], e.w);
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
  // the list: a thread's hits take consecutive places of it in LDS, then it goes out whole
  int hits = 0;
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) hits += bin[k] < list_bins;
  if (hits) {
    int at = atomicAdd(&list_n, hits);
#pragma unroll
    for (int k = 0; k < kPerThread; ++k)
      if (bin[k] < list_bins) list[at++] = make_uint2(i0 + k * kBinThreads, sf_bitcast<uint32_t>(x[k]));
  }
  __syncthreads();
  if ((int)threadIdx.x < list_n)
    o->list[threadIdx.x] = (u64)order_key(sf_bitcast<float>(list[threadIdx.x].y)) << 32 | (uint32_t)~list[threadIdx.x].x;
  if (threadIdx.x == 0) o->list_n = list_n, o->list_bins = list_bins;
}

struct Found {   // a place in a bin's order: the r-th (from 0) of `ties` tokens with this logit
  uint32_t key;
  u64 r, ties;   // (ties: of a search by count)
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
  int cursor[kBins];
  int uncovered;
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
  double per, top, chunk_top;  // (the top that chunks are compared with)
  bool flat;
  const ChunkOut *outs;
  PickSmem &sm;
  int held;  // the bin whose elements lie in sm.el, in order (-1: none)

  __device__ __forceinline__ float at(int i) const {
    const float x = sf_load_as_f32<DT>(logits, row + i);
    return flat ? flat_value(x) : x;
  }
  // f(index, logit) over the row's logits, the loads of eight in flight together
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (int i0 = threadIdx.x; i0 - (int)threadIdx.x < V; i0 += 8 * kSampThreads) {
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = at(min(i0 + k * kSampThreads, V - 1));
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i0 + k * kSampThreads < V) f(i0 + k * kSampThreads, x[k]);
    }
  }
  // The row's elements of the bins first .. last into sm.raw, bin after bin: from the chunks'
  // lists where these have every bin up to `last`. Room has been made by the bins' counts.
  __device__ __forceinline__ void gather(int first, int last) {
    auto put = [&](int bin, u64 e) {
      if (first <= bin && bin <= last) sm.raw[sm.n_before[bin] - sm.n_before[first] + atomicAdd(&sm.cursor[bin], 1)] = e;
    };
    auto clear = [&]() {
      __syncthreads();
      if (threadIdx.x < kBins) sm.cursor[threadIdx.x] = 0;
      if (threadIdx.x == 0) sm.uncovered = 0;
      __syncthreads();
    };
    clear();
    for (int c = threadIdx.x >> 6; c < chunks; c += kSampWaves) {
      const ChunkOut &o = outs[c];
      const double shift = o.top == chunk_top ? 0.0 : chunk_top - o.top;
      const int ln = o.list_n, lane = threadIdx.x & 63;
      const u64 e0 = lane < ln ? o.list[lane] : 0, e1 = lane + 64 < ln ? o.list[lane + 64] : 0;
      if (!(shift <= (double)last)) continue;  // it has nothing there
      if (last - (int)shift >= o.list_bins) sm.uncovered = 1;
      if (lane < ln) put(bin_of(key_value((uint32_t)(e0 >> 32)), per, top).bin, e0);
      if (lane + 64 < ln) put(bin_of(key_value((uint32_t)(e1 >> 32)), per, top).bin, e1);
    }
    __syncthreads();
    if (sm.uncovered) {
      clear();
      // (the bins' range of logits, one bin wider each way, first; then exactly)
      const float from = (float)logit_at(top, last + 2, per), to = (float)logit_at(top, first - 2, per);
      each([&](int i, float x) {
        if (x >= from && x <= to) put(bin_of(x, per, top).bin, (u64)order_key(x) << 32 | (uint32_t)~i);
      });
      __syncthreads();
    }
  }

  __device__ __forceinline__ u64 weight(uint32_t key) const { return bin_of(key_value(key), per, top).w; }
  __device__ __forceinline__ bool in(float x, int bin) const {
    return bin_of(x, per, top).bin == bin;
  }

  // Those elements (n of them) into sm.el in descending order: each counts the larger ones
  // of its bin, eight at a time so that their LDS reads fly together.
  __device__ __forceinline__ void order(int first, int n) {
    if ((int)threadIdx.x < n) {
      const u64 e = sm.raw[threadIdx.x];
      const int bin = bin_of(key_value((uint32_t)(e >> 32)), per, top).bin;
      order_one(e, sm.raw, sm.n_before[bin] - sm.n_before[first], sm.n_before[bin + 1] - sm.n_before[first]);
    }
    __syncthreads();
  }
  // One element of from[lo .. hi) to its place.
  __device__ __forceinline__ void order_one(u64 e, const u64 *from, int lo, int hi) {
    int rank = lo;
    for (int i0 = lo; i0 < hi; i0 += 8) {
      u64 v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = from[min(i0 + j, hi - 1)];
#pragma unroll
      for (int j = 0; j < 8; ++j) rank += i0 + j < hi && v[j] > e;
    }
    sm.el[rank] = e;
  }

  // sm.raw's n elements, of the keys base .. base + 2^bits - 1, into sm.el in order, and their
  // running weights into sm.run: by 256 ranges of keys, then by counting within a range (all
  // of 1000 against each other: 27 us).
  __device__ __forceinline__ void order_keys(uint32_t base, int bits, int n) {
    const int lane = threadIdx.x, shift = max(bits - 8, 0);
    const bool own = (int)threadIdx.x < n;
    const u64 e = own ? sm.raw[threadIdx.x] : 0;
    const int part = own ? 255 - (int)(((uint32_t)(e >> 32) - base) >> shift) : 0;
    __syncthreads();
    if (threadIdx.x < 256) sm.cursor[threadIdx.x] = 0;
    __syncthreads();
    const int slot = own ? atomicAdd(&sm.cursor[part], 1) : 0;
    __syncthreads();
    if (threadIdx.x < 64) {
      int c[4], run = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) run += c[j] = sm.cursor[4 * lane + j];
      const int sum = run;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(run, off, 64);
        if (lane >= off) run += o;
      }
      run -= sum;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sm.hist[4 * lane + j] = run;
        run += c[j];
      }
    }
    __syncthreads();
    const int lo = (int)sm.hist[part], hi = lo + sm.cursor[part];
    if (own) sm.run[lo + slot] = e;
    __syncthreads();
    if (own) order_one(e, sm.run, lo, hi);
    __syncthreads();
    scan(n);
  }
  // The range of keys of a bin, two bins wider each way.
  __device__ __forceinline__ void keys_of(int bin, uint32_t &base, int &bits) const {
    base = order_key((float)logit_at(top, bin + 2, per));
    bits = 32 - __clz((int)((order_key((float)logit_at(top, bin - 2, per)) - base) | 1));
  }

  // The elements of a bin of at most kBinCap into sm.el in order, running weights into sm.run.
  __device__ __forceinline__ void hold(int bin) {
    if (held == bin) return;
    held = bin;
    uint32_t base;
    int bits;
    keys_of(bin, base, bits);
    gather(bin, bin);
    order_keys(base, bits, sm.n[bin]);
  }
  // a wave's scan, then the waves before it
  __device__ __forceinline__ void scan(int n) {
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
  __device__ __forceinline__ Found find(int bin, double x, bool by_count) {
    int n = sm.n[bin];
    const u64 all = by_count ? (u64)n : sm.w[bin];
    u64 target = x >= (double)all ? all - 1 : x > 0 ? (u64)x : 0;
    u64 above_w = 0;
    if (n <= kBinCap) {
      hold(bin);
    } else {
      // The range of keys that the target falls into, 256 parts of it a pass over the row
      // (highest first: their counts and weights), until a part's elements can be ordered
      // or it is a single key.
      held = -1;
      uint32_t base;  // keys base .. base + 2^bits - 1
      int bits;
      keys_of(bin, base, bits);
#pragma unroll 1
      do {
        const int shift = max(bits - 8, 0);
        __syncthreads();
        if (threadIdx.x < 256) sm.hist[threadIdx.x] = 0, sm.cursor[threadIdx.x] = 0;
        __syncthreads();
        each([&](int, float v) {
          const uint32_t k = order_key(v) - base;
          if ((u64)k >> bits == 0) {
            const Binned e = bin_of(v, per, top);
            if (e.bin == bin) {
              atomicAdd(&sm.hist[255 - (k >> shift)], e.w);
              atomicAdd(&sm.cursor[255 - (k >> shift)], 1);
            }
          }
        });
        __syncthreads();
        if (threadIdx.x < 64) {  // lane l: parts 4 l .. 4 l + 3
          const int lane = threadIdx.x;
          u64 w = 0, c = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            w += sm.hist[4 * lane + j];
            c += sm.cursor[4 * lane + j];
          }
          u64 w_run = w, c_run = c;
#pragma unroll
          for (int off = 1; off < 64; off <<= 1) {
            const u64 ow = __shfl_up(w_run, off, 64), oc = __shfl_up(c_run, off, 64);
            if (lane >= off) {
              w_run += ow;
              c_run += oc;
            }
          }
          w_run -= w;
          c_run -= c;
          for (int j = 4 * lane; j < 4 * lane + 4; ++j) {
            const u64 wj = sm.hist[j], cj = sm.cursor[j];
            const u64 before = by_count ? c_run : w_run;
            if (before <= target && target < before + (by_count ? cj : wj)) {
              sm.tmp[0] = j;
              sm.tmp[1] = w_run;
              sm.tmp[2] = c_run;
            }
            w_run += wj;
            c_run += cj;
          }
        }
        __syncthreads();
        const int part = (int)sm.tmp[0];
        base += (uint32_t)(255 - part) << shift;
        bits = shift;
        above_w += sm.tmp[1];
        target -= by_count ? sm.tmp[2] : sm.tmp[1];
        n = sm.cursor[part];
      } while (n > kBinCap && bits > 0);
      if (n > kBinCap) {  // ties alone
        const u64 w = weight(base), r = by_count ? target : target / w;
        return Found{base, r, (u64)n, above_w + (r + 1) * w, -1};
      }
      __syncthreads();
      if (threadIdx.x == 0) sm.cursor[0] = 0;
      __syncthreads();
      each([&](int i, float v) {
        const uint32_t k = order_key(v);
        if ((u64)(k - base) >> bits == 0 && in(v, bin)) sm.raw[atomicAdd(&sm.cursor[0], 1)] = (u64)k << 32 | (uint32_t)~i;
      });
      __syncthreads();
      order_keys(base, bits, n);
    }
    const int t = threadIdx.x;
    const bool over = t < n && (by_count ? (u64)(t + 1) : sm.run[t]) > target;
    const int passed = (int)block_sum(t < n && !over, sm);
    const int j = min(passed, n - 1);
    const uint32_t key = (uint32_t)(sm.el[j] >> 32);
    const bool tie = t < n && (uint32_t)(sm.el[t] >> 32) == key;
    const u64 c = block_sum((u64)tie << 32 | (tie && t < j), sm);
    return Found{key, c & 0xffffffffu, c >> 32, above_w + sm.run[j], (int)~(uint32_t)sm.el[j]};
  }

  // Weight of the bin's tokens that weigh at least `least` of the largest.
  __device__ __forceinline__ u64 heavy(int bin, double M, double inv_t, uint32_t kmax, double least) {
    auto is = [&](uint32_t k) {
      return k == kmax || exp(((double)key_value(k) - M) * inv_t) >= least;
    };
    u64 s = 0;
    if (sm.n[bin] <= kBinCap) {
      hold(bin);
      if ((int)threadIdx.x < sm.n[bin]) {
        const uint32_t k = (uint32_t)(sm.el[threadIdx.x] >> 32);
        s = is(k) ? weight(k) : 0;
      }
    } else {
      each([&](int, float v) {
        if (in(v, bin) && is(order_key(v))) s += bin_of(v, per, top).w;
      });
    }
    return block_sum(s, sm);
  }

  // The index of the r-th token with this logit.
  __device__ __forceinline__ int index_of(uint32_t key, u64 r) {
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

  // The first bin at which `is` holds (it holds from there on), kBins where none: every
  // wave finds it by itself.
  template <class Is>
  __device__ __forceinline__ int first_bin(Is is) const {
    const int lane = threadIdx.x & 63;
    int n = 0;
#pragma unroll
    for (int j = 0; j < kBins / 64; ++j) n += __popcll(__ballot(!is(lane + 64 * j)));
    return n;
  }
  // The first bin up to `last` whose weight, with that of the bins before it, exceeds x.
  __device__ __forceinline__ int bin_past(double x, int last) const {
    return min(first_bin([&](int t) { return sm.before[t + 1] > x; }), last);
  }
  // ln of a token's share of `total`.
  __device__ __forceinline__ float logprob(uint32_t key, uint32_t kmax, double M, double inv_t, double total) const {
    return (float)((key == kmax ? 0.0 : ((double)key_value(key) - M) * inv_t) -
                   log(total / ((double)weight(kmax) * sm.fac[0])));
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
  // the chunks' bins and lists are on their way before the maximum says where they belong
  constexpr int kAhead = 8, kParts = kSampThreads / kBins;  // (32 chunks: 262144 tokens)
  const int my_bin = threadIdx.x & (kBins - 1), part = threadIdx.x / kBins;
  u64 v[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    const int c = part + j * kParts;
    v[j] = c < chunks ? o[c].bins[my_bin] : 0;
  }
  u64 best = 0;
  for (int c = lane; c < chunks; c += 64) best = o[c].best > best ? o[c].best : best;
  if (threadIdx.x < kBins) sm.w[threadIdx.x] = 0, sm.n[threadIdx.x] = 0;
  best = wave_max(best);
  __syncthreads();
  uint32_t kmax = (uint32_t)(best >> 32);
  const float T = rp.t(b);
  const bool empty = kmax == kNoKey;
  if (empty || !(T > 0.f)) {
    if (threadIdx.x == 0) {
      tokens[b] = empty ? -1 : (int)~(uint32_t)best;
      if (rp.hist) rp.hist[rp.place(b)] = empty ? -1 : (int)~(uint32_t)best;
      if (logprobs) logprobs[b] = empty ? -INFINITY : 0.f;
    }
    return;
  }
  const bool flat = key_value(kmax) == INFINITY;
  if (flat) kmax = order_key(0.f);
  const double M = (double)key_value(kmax), inv_t = fmax(1.0 / (double)T, 1e-300), per = bins_per_logit(T);
  Row<DT> row = {logits, (size_t)b * row_stride, V, chunks, per, top_bin((float)M, per), 0, flat, o, sm, -1};
  row.chunk_top = flat ? INFINITY : row.top;
  // the row's bins (whole numbers: the order of the additions changes nothing)
  for (int c = part, j = 0; c < chunks; c += kParts, ++j) {
    const double shift = o[c].top == row.chunk_top ? 0.0 : row.chunk_top - o[c].top;
    u64 e = j < kAhead ? 0 : o[c].bins[my_bin];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) e = i == j ? v[i] : e;
    if (e && shift < (double)(kBins - my_bin)) {
      atomicAdd(&sm.w[my_bin + (int)shift], e & kWeightMask);
      atomicAdd(&sm.n[my_bin + (int)shift], (int)(e >> kCountShift));
    }
  }
  if (threadIdx.x < kBins) sm.fac[threadIdx.x] = exp(-kDelta * (int)threadIdx.x) * 0x1p-36;
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
  const int k = rp.top_ks ? rp.top_ks[b] : rp.top_k;
  const float tp = rp.top_ps ? rp.top_ps[b] : rp.top_p, mp = rp.min_ps ? rp.min_ps[b] : rp.min_p;
  const int place = rp.place(b);
  const double uu = fmin(fmax((double)u[place], 0.0), 1.0), least = fmin((double)mp, 1.0);
  const bool by_k = k > 0 && k < sm.n_before[kBins], by_p = tp < 1.f, by_m = mp > 0.f;
  int m_bin = kBins;  // the bin of the least weight that min-p leaves
  if (by_m) {
    const double below = row.top - floor(axis_of((float)M, per) + log(least) * (1.0 / kDelta));
    m_bin = below < (double)kBins ? max(0, (int)below) : kBins;
  }
  // The head: the bins up to the end of what the filters leave. top-p's share is of what
  // top-k left, so where both are set the head reaches to the k-th token.
  const int k_bin = by_k ? row.first_bin([&](int t) { return sm.n_before[t + 1] >= k; }) : kBins - 1;
  int head = k_bin;
  if (!by_k) {
    const double x = by_p ? fmax((double)tp, 0.0) * sm.before[kBins] : by_m ? sm.before[kBins] : uu * sm.before[kBins];
    head = min(row.bin_past(x, kBins - 1), m_bin);
  }
  if (sm.n_before[head + 1] <= kHeadCap) {
    const int n = sm.n_before[head + 1];
    row.gather(0, head);
    row.order(0, n);
    if (threadIdx.x >= 64) return;
    // lane l: the places P l .. P l + P - 1 of the order
    constexpr int P = kHeadCap / 64;
    uint32_t key[P];
    double w[P], upto[P], sum = 0;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int i = P * lane + j;
      key[j] = i < n ? (uint32_t)(sm.el[i] >> 32) : 0;
      const Binned e = bin_of(key_value(key[j]), per, row.top);
      w[j] = i < n ? (double)e.w * sm.fac[min(e.bin, kBins - 1)] : 0.0;
      sum += w[j];
    }
    double run = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double v = __shfl_up(run, off, 64);
      if (lane >= off) run += v;
    }
    double before = __shfl_up(run, 1, 64);
    if (lane == 0) before = 0;
#pragma unroll
    for (int j = 0; j < P; ++j) upto[j] = j == P - 1 ? run : (j ? upto[j - 1] : before) + w[j];
    // how many places, from the first on, a condition holds at; a value at a place
    auto count = [&](auto is) {
      int c = 0;
#pragma unroll
      for (int j = 0; j < P; ++j) c += __popcll(__ballot(P * lane + j < n && is(j)));
      return c;
    };
    auto upto_at = [&](int i) {
      double v = 0;
#pragma unroll
      for (int j = 0; j < P; ++j)
        if (i % P == j) v = upto[j];
      return __shfl(v, i / P, 64);
    };
    int kept = n;
    double total = sm.before[kBins];
    if (by_k) {
      const uint32_t kth = (uint32_t)(sm.el[k - 1] >> 32);
      kept = count([&](int j) { return key[j] >= kth; });
      total = upto_at(kept - 1);
    }
    if (by_p) {
      const double bound = fmax((double)tp, 0.0) * total;
      kept = min(kept, count([&](int j) { return (j ? upto[j - 1] : before) <= bound; }));
    }
    if (by_m)
      kept = min(kept, count([&](int j) { return key[j] == kmax || exp(((double)key_value(key[j]) - M) * inv_t) >= least; }));
    kept = max(kept, 1);
    if (by_k || by_p || by_m) total = upto_at(kept - 1);
    const double target = uu * total;
    const int at = min(count([&](int j) { return upto[j] <= target; }), kept - 1);
    if (lane == 0) {
      const u64 e = sm.el[at];
      tokens[b] = (int)~(uint32_t)e;
      if (rp.hist) rp.hist[place] = (int)~(uint32_t)e;
      if (logprobs) logprobs[b] = row.logprob((uint32_t)(e >> 32), kmax, M, inv_t, total);
    }
    return;
  }
  // What stays: the bins before `last`, and of that bin the tokens before and with the
  // (r + 1)-th that has the logit `key`: `upto` of weight. At first everything.
  int last = kBins - 1;
  uint32_t key = 0;
  u64 r = ~0ull >> 1, upto = sm.w[kBins - 1];
  auto weight_kept = [&]() { return sm.before[last] + (double)upto * sm.fac[last]; };
  double total = 0;
  Found f;
#pragma unroll 1  // (one copy of the search: the code of four costs more than the jumps)
  for (int stage = 0; stage < 4; ++stage) {
    int bin = k_bin;
    double x = 0;
    if (stage == 0) {  // top-k
      if (!by_k) continue;
      x = (double)(k - 1 - sm.n_before[bin]);
    } else if (stage == 2) {  // min-p: those that weigh enough, all before any other
      if (!by_m || m_bin > last) continue;
      const u64 w = row.heavy(m_bin, M, inv_t, kmax, least);
      if (m_bin < last || w < upto) {
        last = m_bin;
        upto = w;
      }
      continue;
    } else {  // top-p's end, then the draw
      if (stage == 1 && !by_p) continue;
      total = weight_kept();
      const double target = (stage == 1 ? fmax((double)tp, 0.0) : uu) * total;
      bin = row.bin_past(target, last);
      // (an empty bin, by the prefix sums' rounding, or a last one of which nothing stays:
      // the last token before it)
      while (bin > 0 && (bin == last ? upto == 0 : sm.w[bin] == 0)) --bin;
      x = (target - sm.before[bin]) / sm.fac[bin];
      const double most = (double)(bin == last ? upto : sm.w[bin]);
      if (!(x < most)) x = most - 1.0;
    }
    f = row.find(bin, x, stage == 0);
    if (stage == 0) {  // the ties of the k-th stay too
      last = bin;
      key = f.key;
      upto = f.upto + (f.ties - 1 - f.r) * row.weight(key);
      r = f.ties - 1;
    } else if (stage == 1 && (bin < last || f.key > key || (f.key == key && f.r < r))) {
      last = bin;
      key = f.key;
      r = f.r;
      upto = f.upto;
    }
  }
  const int token = f.index >= 0 ? f.index : row.index_of(f.key, f.r);
  if (threadIdx.x == 0) {
    tokens[b] = token;
    if (rp.hist) rp.hist[place] = token;
    if (logprobs) logprobs[b] = row.logprob(f.key, kmax, M, inv_t, total);
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
                         float *logprobs, const int32_t *at, int at_add, int u_n, int32_t *hist, void *workspace, size_t workspace_bytes, void *stream) {
  SF_REQUIRE(B >= 0 && V > 0, SF_EINVAL, "invalid sampling shape B=%d V=%d", B, V);
  SF_REQUIRE(V <= (1 << 24), SF_EUNSUPPORTED, "V=%d: at most 16777216 tokens", V);
  SF_REQUIRE(dtype >= SF_F32 && dtype <= SF_BF16, SF_EINVAL, "bad dtype %d", dtype);
  SF_REQUIRE(row_stride >= 0, SF_EINVAL, "row stride %lld", row_stride);
  SF_REQUIRE(temperature == temperature && top_k >= 0 && top_p > 0.f && min_p >= 0.f && min_p <= 1.f, SF_EINVAL,
             "need top_k >= 0, top_p > 0, 0 <= min_p <= 1 (got %d, %g, %g; temperature %g)", top_k, top_p, min_p,
             temperature);
  if (B == 0) return SF_OK;
  SF_REQUIRE(logits && u && tokens, SF_EINVAL, "null pointer argument");
  SF_REQUIRE(at ? u_n >= B : !hist, SF_EINVAL, at ? "%d numbers for %d rows" : "hist without at", u_n, B);
  const long long chunks = sample_chunks(V);
  SF_REQUIRE(B * chunks <= 0x7fffffffLL, SF_EINVAL, "B=%d rows of %d exceed the grid", B, V);
  SF_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0, SF_EINVAL, "workspace must be 256-byte aligned");
  const size_t need = sf_sample_workspace_bytes(B, V);
  SF_REQUIRE(workspace_bytes >= need, SF_EINVAL, "sampling workspace too small: %zu < %zu", workspace_bytes, need);
  const RowParams rp = {temperature, top_p, min_p, top_k, temperatures, top_ps, min_ps, top_ks, at, hist, at_add, u_n, B};
  ChunkOut *outs = (ChunkOut *)workspace;
  hipStream_t st = (hipStream_t)stream;
#define SF_SAMP(DT)                                                                                                \
  do {                                                                                                             \
    k_sample_bins<DT><<<(unsigned)(B * chunks), kBinThreads, 0, st>>>(logits, row_stride, V, (int)chunks, rp, outs); \
    k_sample_pick<DT><<<B, kSampThreads, 0, st>>>(logits, row_stride, V, (int)chunks, u, rp, outs, tokens, logprobs); \
  } while (0)
  if (dtype == SF_F32) SF_SAMP(SF_F32);
  else if (dtype == SF_F16) SF_SAMP(SF_F16);
  else SF_SAMP(SF_BF16);
#undef SF_SAMP
  return sf_check_launch("sf_sample");
}
