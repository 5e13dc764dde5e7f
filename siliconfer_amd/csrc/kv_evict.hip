// kv_evict.hip — a bounded KV cache: the slots with the least accumulated attention
// weight leave it (gfx950).
//
// Of the n = lengths[b] slots of a (sequence, kv head) the `budget` with the largest
// keys stay. A slot's key is its score, but slots of the newest `recent` tokens
// (positions[slot] >= seen[b] - recent) come before every score, a NaN score counts
// as -inf, and equal keys go to the lower slot. Attention does not depend on the
// order of the slots (keys are rotated before they are cached), so the kept slots
// behind the budget move into the holes below it, both in ascending order: sources
// and destinations are apart, every copy is independent of the others, and the
// least is moved.
//
// k_evict_select: one workgroup a (sequence, kv head), up to 12288 keys in LDS. The
// threshold t is the largest key that `budget` slots reach: radix selection, 11 + 11 + 10
// bits, each a histogram of counts in LDS (integer atomics: their order changes nothing)
// and a scan of it from the top; the newest tokens' slots are counted by ballots and left
// out of it. Then the (hole, donor) list by ballots over the waves' segments. Few moves
// are made by the same workgroup, many by a second launch over every CU.
// Bound by the latency of its dozen barriers and of one read of scores and positions:
// 7.8 us for 2 heads of 1088 slots, moves among them, 13.3 + 7.4 for 32 heads of up to 8191
// cut to 2048 (a search of the threshold bit pair by bit pair with counts over the
// workgroup, keys in registers: 13.4 + 4.0 and 88 + 6.6; keys read again each time: 25 and 71).
#include "sf_common.h"

namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kMoveThreads = 256;

// Order-preserving bits of a score; kProtected for the newest tokens' slots.
constexpr uint32_t kProtected = 0xffffffffu;
__device__ __forceinline__ uint32_t evict_key(float score, int position, long long first_recent) {
  if ((long long)position >= first_recent) return kProtected;
  float f = score != score ? -INFINITY : score;
  f = f == 0.f ? 0.f : f;  // -0 is +0
  const uint32_t u = sf_bitcast<uint32_t>(f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The sum of v over the waves before this one, and over all of them.
__device__ __forceinline__ int waves_before(int v, int *cnt, int *total) {
  __syncthreads();
  if ((threadIdx.x & 63) == 0) cnt[threadIdx.x >> 6] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) {
    before += w < (int)(threadIdx.x >> 6) ? cnt[w] : 0;
    all += cnt[w];
  }
  *total = all;
  return before;
}

struct EvictArgs {
  int8_t *kc, *vc;
  void *ks, *vs;
  float *scores;
  int *positions;
  const int *lengths, *seen;
  int *lengths_out, *counts;
  int2 *pairs;
  int T, seen_host, budget, recent, max_moves, KVH, T_cap, D;
  int wide, scale_bytes;  // 16-byte pieces of codes, else 8; 2 or 4
  int moves;              // the selecting workgroup moves its pairs itself
};

// Copies a head's n pairs, items first, first + step, ...: the codes in pieces of VB bytes
// (a pair's K, then its V), then the pairs' scales, scores and positions.
template <int VB>
__device__ void move_pairs(const EvictArgs &a, int bh, int n, const int2 *list, uint32_t first, uint32_t step) {
  const uint32_t half = a.D / VB, per = 2 * half, items = (uint32_t)n * per;  // (2^20 pairs of 64 at most)
  const size_t row0 = (size_t)bh * a.T_cap;
#pragma unroll 4
  for (uint32_t e = first; e < items; e += step) {
    const uint32_t m = e / per, i = e - m * per;
    const int2 mv = list[m];
    int8_t *c = i < half ? a.kc : a.vc;
    const size_t at = (size_t)(i < half ? i : i - half) * VB, to = (row0 + mv.x) * a.D + at, from = (row0 + mv.y) * a.D + at;
    if constexpr (VB == 16) *(u32x4 *)(c + to) = *(const u32x4 *)(c + from);
    else *(u32x2 *)(c + to) = *(const u32x2 *)(c + from);
  }
  for (uint32_t m = first; m < (uint32_t)n; m += step) {
    const size_t to = row0 + list[m].x, from = row0 + list[m].y;
    if (a.scale_bytes == 2) {
      const uint16_t k = ((const uint16_t *)a.ks)[from], v = ((const uint16_t *)a.vs)[from];
      ((uint16_t *)a.ks)[to] = k;
      ((uint16_t *)a.vs)[to] = v;
    } else {
      const uint32_t k = ((const uint32_t *)a.ks)[from], v = ((const uint32_t *)a.vs)[from];
      ((uint32_t *)a.ks)[to] = k;
      ((uint32_t *)a.vs)[to] = v;
    }
    const float f = a.scores[from];
    const int p = a.positions[from];
    a.scores[to] = f;
    a.positions[to] = p;
  }
}

// KEYS: keys held in LDS (0: read again from memory on every pass; held in registers, 32 a
// thread, the unrolled passes outgrew the instruction cache: 24 us where LDS takes 14.2).
// Wave w has the slots from w 64 steps on, step r's lane l slot w 64 steps + 64 r + l,
// so that an ascending order over slots is one over (wave, r, lane).
template <int KEYS>
__global__ void __launch_bounds__(kSelThreads)
k_evict_select(EvictArgs a) {
  constexpr int kDigits = 2048;
  __shared__ uint32_t keys[KEYS ? KEYS : 1];
  __shared__ int hist[kDigits];
  __shared__ int cnt[kSelWaves];
  __shared__ int found[3];
  const int h = blockIdx.x, b = blockIdx.y, bh = b * a.KVH + h, budget = a.budget;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = max(0, min(a.lengths ? a.lengths[b] : a.T, a.T_cap));
  if (h == 0 && threadIdx.x == 0) a.lengths_out[b] = min(n, budget);
  if (n <= budget) {
    if (threadIdx.x == 0) a.counts[bh] = 0;
    return;
  }
  const long long first_recent = (long long)(a.seen ? a.seen[b] : a.seen_host) - a.recent;
  const float *sc = a.scores + (size_t)bh * a.T_cap;
  const int *ps = a.positions + (size_t)bh * a.T_cap;
  const int steps = (n + kSelThreads - 1) / kSelThreads;
  const int lo = min(wave * 64 * steps, n), hi = min(lo + 64 * steps, n);
  constexpr int U = 4;  // steps whose loads fly together
  // each(f): f(the step's first slot, in range?, key) over the wave's slots in order
  auto each = [&](auto f) {
    for (int i0 = lo; i0 < hi; i0 += 64 * U) {
      uint32_t k[U];
      if constexpr (KEYS != 0) {  // (a wave reads only what it wrote itself)
#pragma unroll
        for (int u = 0; u < U; ++u) k[u] = keys[min(i0 + 64 * u + lane, n - 1)];
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = min(i0 + 64 * u + lane, n - 1);
          k[u] = evict_key(sc[i], ps[i], first_recent);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + 64 * u < hi) f(i0 + 64 * u, i0 + 64 * u + lane < hi, k[u]);
    }
  };
  // the newest tokens counted, the others' highest digits into the histogram
  hist[threadIdx.x] = 0;
  hist[threadIdx.x + kSelThreads] = 0;
  __syncthreads();
  int newest = 0, n_newest;
  for (int i0 = lo; i0 < hi; i0 += 64 * U) {
    float f[U];
    int p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + 64 * u + lane, n - 1);
      f[u] = sc[i];
      p[u] = ps[i];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + 64 * u + lane;
      const uint32_t k = evict_key(f[u], p[u], first_recent);
      if (KEYS != 0 && i < hi) keys[KEYS ? i : 0] = k;
      newest += __popcll(__ballot(i < hi && k == kProtected));
      if (i < hi && k != kProtected) atomicAdd(&hist[k >> 21], 1);
    }
  }
  waves_before(newest, cnt, &n_newest);  // (a barrier: the histogram is whole)
  // t: the key from which on slots stay; of the n_ties with (at least) its digits `stay` do
  uint32_t t = kProtected;
  int stay = budget, n_ties = n_newest;
  if (n_newest < budget) {
    uint32_t prefix = 0, mask = 0;
    stay = budget - n_newest;
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t digits = pass == 2 ? 1023u : 2047u;
      if (pass) {
        hist[threadIdx.x] = 0;
        hist[threadIdx.x + kSelThreads] = 0;
        __syncthreads();
        each([&](int, bool in, uint32_t k) {
          if (in && k != kProtected && (k & mask) == prefix) atomicAdd(&hist[k >> shift & digits], 1);
        });
        __syncthreads();
      }
      // thread i: digits 2047 - 2 i and 2046 - 2 i
      const int2 own = ((const int2 *)hist)[kSelThreads - 1 - threadIdx.x];
      int run = own.x + own.y;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int v = __shfl_up(run, off, 64);
        if (lane >= off) run += v;
      }
      int all;
      run += waves_before(__shfl(run, 63, 64), cnt, &all);
      const int before = run - own.x - own.y;
      if (before < stay && stay <= run) {
        const bool high = stay <= before + own.y;
        found[0] = 2047 - 2 * (int)threadIdx.x - !high;
        found[1] = high ? before : before + own.y;
        found[2] = high ? own.y : own.x;
      }
      __syncthreads();
      prefix |= (uint32_t)found[0] << shift;
      mask |= digits << shift;
      stay -= found[1];
      n_ties = found[2];
      if (n_ties == stay) break;  // every key from this digit on stays: no lower digits to find
    }
    t = prefix;
  }
  const unsigned long long below = (1ull << lane) - 1;
  int tie0 = 0;
  const bool all_ties = n_ties == stay;  // (distinct scores: no ranks to find)
  if (!all_ties) {
    int ties = 0, total;
    each([&](int, bool in, uint32_t k) { ties += __popcll(__ballot(in && k == t)); });
    tie0 = waves_before(ties, cnt, &total);
  }
  // the wave's holes and donors, counted, then listed
  int seen_ties = tie0, holes = 0, donors = 0;
  auto sort_out = [&](int i0, bool in, uint32_t k, unsigned long long *hole, unsigned long long *donor) {
    bool stays = in && k >= t;
    if (!all_ties) {
      const unsigned long long tie = __ballot(in && k == t);
      stays = in && (k > t || (k == t && seen_ties + __popcll(tie & below) < stay));
      seen_ties += __popcll(tie);
    }
    *hole = __ballot(in && !stays && i0 + lane < budget);
    *donor = __ballot(stays && i0 + lane >= budget);
  };
  each([&](int i0, bool in, uint32_t k) {
    unsigned long long hole, donor;
    sort_out(i0, in, k, &hole, &donor);
    holes += __popcll(hole);
    donors += __popcll(donor);
  });
  int n_holes, n_donors;
  int at = waves_before(holes, cnt, &n_holes), from = waves_before(donors, cnt, &n_donors);
  if (threadIdx.x == 0) a.counts[bh] = n_holes;
  seen_ties = tie0;
  int2 *list = a.pairs + (size_t)bh * a.max_moves;
  each([&](int i0, bool in, uint32_t k) {
    unsigned long long hole, donor;
    sort_out(i0, in, k, &hole, &donor);
    if (hole >> lane & 1) list[at + __popcll(hole & below)].x = i0 + lane;
    if (donor >> lane & 1) list[from + __popcll(donor & below)].y = i0 + lane;
    at += __popcll(hole);
    from += __popcll(donor);
  });
  if (a.moves) {
    __syncthreads();
    if (a.wide) move_pairs<16>(a, bh, n_holes, list, threadIdx.x, kSelThreads);
    else move_pairs<8>(a, bh, n_holes, list, threadIdx.x, kSelThreads);
  }
}

__global__ void __launch_bounds__(kMoveThreads) k_evict_move(EvictArgs a) {
  const int bh = blockIdx.z * a.KVH + blockIdx.y;
  const int2 *list = a.pairs + (size_t)bh * a.max_moves;
  const long long first = (long long)blockIdx.x * kMoveThreads + threadIdx.x, step = (long long)gridDim.x * kMoveThreads;
  if (a.wide) move_pairs<16>(a, bh, a.counts[bh], list, first, step);
  else move_pairs<8>(a, bh, a.counts[bh], list, first, step);
}

}  // namespace

// A pair's slots lie on both sides of the budget, so a head has at most this many.
static int evict_max_moves(int budget, int T_max) {
  const int over = T_max > budget ? T_max - budget : 0;
  return budget < over ? budget : over;
}

extern "C" size_t sf_kv_evict_workspace_bytes(int B, int KVH, int budget, int T_max) {
  if (B <= 0 || KVH <= 0 || budget <= 0 || T_max < 0) return 0;
  const size_t n = (size_t)B * KVH;
  return sf_align256(n * sizeof(int)) + n * evict_max_moves(budget, T_max) * sizeof(int2);
}

extern "C" int sf_kv_evict(int8_t *k_codes, void *k_scales, int8_t *v_codes, void *v_scales, int scale_dtype,
                           float *scores, int32_t *positions, const int32_t *lengths, int T,
                           const int32_t *seen, int seen_host, int budget, int recent, int32_t *lengths_out,
                           void *workspace, size_t workspace_bytes, int B, int KVH, int T_cap, int D,
                           void *stream) {
  SF_REQUIRE(B > 0 && KVH > 0 && T_cap > 0 && D > 0, SF_EINVAL, "invalid KV shape B=%d KVH=%d T_cap=%d D=%d", B,
             KVH, T_cap, D);
  SF_REQUIRE(D % 8 == 0 && D <= 256, SF_EUNSUPPORTED, "head_dim=%d: need D %% 8 == 0 and D <= 256", D);
  SF_REQUIRE(scale_dtype == SF_F16 || scale_dtype == SF_F32, SF_EINVAL, "bad scale dtype %d", scale_dtype);
  SF_REQUIRE(budget > 0 && recent >= 0 && recent <= budget, SF_EINVAL,
             "need budget > 0 and 0 <= recent <= budget (got %d, %d)", budget, recent);
  SF_REQUIRE(lengths || (T >= 0 && T <= T_cap), SF_EINVAL, "%d slots of a capacity of %d", T, T_cap);
  SF_REQUIRE(T_cap < (1 << 21), SF_EUNSUPPORTED, "capacity %d: at most 2097151 slots", T_cap);
  SF_REQUIRE(KVH <= 65535 && B <= 65535, SF_EINVAL, "B=%d KVH=%d exceed the grid", B, KVH);
  SF_REQUIRE(k_codes && k_scales && v_codes && v_scales && scores && positions && lengths_out, SF_EINVAL,
             "null pointer argument");
  SF_REQUIRE(lengths_out != lengths, SF_EINVAL, "lengths_out must not be lengths");
  SF_REQUIRE((((uintptr_t)k_codes | (uintptr_t)v_codes) & 7) == 0, SF_EINVAL,
             "KV code buffers must be 8-byte aligned");
  const int T_max = lengths ? T_cap : T, most = evict_max_moves(budget, T_max);
  const size_t need = sf_kv_evict_workspace_bytes(B, KVH, budget, T_max);
  SF_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0, SF_EINVAL, "workspace must be 16-byte aligned");
  SF_REQUIRE(workspace_bytes >= need, SF_EINVAL, "eviction workspace too small: %zu < %zu", workspace_bytes, need);
  int *counts = (int *)workspace;
  int2 *pairs = (int2 *)((char *)workspace + sf_align256((size_t)B * KVH * sizeof(int)));
  hipStream_t st = (hipStream_t)stream;
  const int wide = D % 16 == 0 && (((uintptr_t)k_codes | (uintptr_t)v_codes) & 15) == 0;
  // Moved by the selecting workgroup up to 96 KB a head (us in one launch / two, moves of
  // every head to choose: 2 heads of 8 KB 7.6 / 9.3, 32 of 67 KB 9.8 / 10.4, 32 of 134 KB
  // 12.5 / 12.7, 8 of 134 KB 12.0 / 11.5, 32 of 268 KB 15.3 / 15.0, 32 of 1.6 MB 30.7 / 21.2).
  const int moves = (long long)most * (2 * D + 12) <= 96 << 10;
  const EvictArgs a = {k_codes, v_codes, k_scales, v_scales, scores, positions, lengths, seen, lengths_out, counts,
                       pairs, T, seen_host, budget, recent, most, KVH, T_cap, D, wide,
                       scale_dtype == SF_F16 ? 2 : 4, moves};
  const dim3 heads(KVH, B);
  if (T_max <= 2048) k_evict_select<2048><<<heads, kSelThreads, 0, st>>>(a);
  else if (T_max <= 12288) k_evict_select<12288><<<heads, kSelThreads, 0, st>>>(a);
  else if (T_max <= 32768) k_evict_select<32768><<<heads, kSelThreads, 0, st>>>(a);
  else k_evict_select<0><<<heads, kSelThreads, 0, st>>>(a);
  if (most && !moves) {
    const long long blocks = ((long long)most * (2 * (D / (wide ? 16 : 8)) + 1) + kMoveThreads - 1) / kMoveThreads;
    k_evict_move<<<dim3((unsigned)(blocks < 64 ? blocks : 64), KVH, B), kMoveThreads, 0, st>>>(a);
  }
  return sf_check_launch("sf_kv_evict");
}
