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
// k_evict_select: one workgroup a (sequence, kv head). The threshold t is the
// largest key that `budget` slots reach, found two bits at a time from the top
// (three counts a step, packed in one 64-bit sum: no atomics). Then t's ties by
// ascending slot and the (hole, donor) list by ballots over the waves' segments.
// k_evict_move copies the list's pairs: codes, scales, scores, positions.
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

// Sum over the workgroup; every thread gets it. `red` holds one value a wave.
__device__ __forceinline__ unsigned long long block_sum(unsigned long long v, unsigned long long *red) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();  // the previous sum has been read
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  unsigned long long s = 0;
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) s += red[w];
  return s;
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

__global__ void __launch_bounds__(kSelThreads)
k_evict_select(const float *__restrict__ scores, const int *__restrict__ positions,
               const int *__restrict__ lengths, int T, const int *__restrict__ seen, int seen_host, int budget,
               int recent, int *__restrict__ lengths_out, int *__restrict__ counts, int2 *__restrict__ pairs,
               int max_moves, int KVH, int T_cap) {
  __shared__ unsigned long long red[kSelWaves];
  __shared__ int cnt[kSelWaves];
  const int h = blockIdx.x, b = blockIdx.y, bh = b * KVH + h;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = max(0, min(lengths ? lengths[b] : T, T_cap));
  if (h == 0 && threadIdx.x == 0) lengths_out[b] = min(n, budget);
  if (n <= budget) {
    if (threadIdx.x == 0) counts[bh] = 0;
    return;
  }
  const long long first_recent = (long long)(seen ? seen[b] : seen_host) - recent;
  const float *sc = scores + (size_t)bh * T_cap;
  const int *ps = positions + (size_t)bh * T_cap;
  auto key = [&](int i) { return evict_key(sc[i], ps[i], first_recent); };
  uint32_t t = 0;
  for (int shift = 30; shift >= 0; shift -= 2) {
    const uint32_t c1 = t | (1u << shift), c2 = t | (2u << shift), c3 = t | (3u << shift);
    unsigned long long c = 0;  // three counts of 21 bits
    for (int i = threadIdx.x; i < n; i += kSelThreads) {
      const uint32_t k = key(i);
      c += (k >= c1 ? 1ull : 0ull) | (k >= c2 ? 1ull << 21 : 0ull) | (k >= c3 ? 1ull << 42 : 0ull);
    }
    c = block_sum(c, red);
    const int n1 = (int)(c & 0x1fffff), n2 = (int)(c >> 21 & 0x1fffff), n3 = (int)(c >> 42);
    t = n3 >= budget ? c3 : n2 >= budget ? c2 : n1 >= budget ? c1 : t;
  }
  // ties of t that stay: the first `stay` of them by slot
  const int per = ((n + kSelWaves - 1) / kSelWaves + 63) & ~63;  // a wave's slots
  const int lo = min(wave * per, n), hi = min(lo + per, n);
  int above = 0, ties = 0;
  for (int i0 = lo; i0 < hi; i0 += 64) {
    const uint32_t k = i0 + lane < hi ? key(i0 + lane) : 0;
    const bool in = i0 + lane < hi;
    above += __popcll(__ballot(in && k > t));
    ties += __popcll(__ballot(in && k == t));
  }
  int n_above, n_ties;
  waves_before(above, cnt, &n_above);
  const int tie0 = waves_before(ties, cnt, &n_ties), stay = budget - n_above;
  int first[2], total[2];
  for (int pass = 0; pass < 2; ++pass) {  // count the wave's holes and donors, then list them
    int seen_ties = tie0, holes = 0, donors = 0;
    for (int i0 = lo; i0 < hi; i0 += 64) {
      const int i = i0 + lane;
      const bool in = i < hi;
      const uint32_t k = in ? key(i) : 0;
      const unsigned long long below = (1ull << lane) - 1, tie = __ballot(in && k == t);
      const bool kept = in && (k > t || (k == t && seen_ties + __popcll(tie & below) < stay));
      const unsigned long long hole = __ballot(in && !kept && i < budget), donor = __ballot(kept && i >= budget);
      if (pass) {
        const int at = first[0] + holes + __popcll(hole & below), from = first[1] + donors + __popcll(donor & below);
        int2 *list = pairs + (size_t)bh * max_moves;
        if (hole >> lane & 1) list[at].x = i;
        if (donor >> lane & 1) list[from].y = i;
      }
      seen_ties += __popcll(tie);
      holes += __popcll(hole);
      donors += __popcll(donor);
    }
    if (!pass) {
      first[0] = waves_before(holes, cnt, &total[0]);
      first[1] = waves_before(donors, cnt, &total[1]);
      if (threadIdx.x == 0) counts[bh] = total[0];
    }
  }
}

// VB bytes a thread (16 or 8): D / VB threads move one pair's K codes, as many its V
// codes, and one thread its scales, score and position.
template <int VB, int SB>
__global__ void __launch_bounds__(kMoveThreads)
k_evict_move(int8_t *__restrict__ kc, void *__restrict__ ks, int8_t *__restrict__ vc, void *__restrict__ vs,
             float *__restrict__ scores, int *__restrict__ positions, const int *__restrict__ counts,
             const int2 *__restrict__ pairs, int max_moves, int KVH, int T_cap, int D) {
  const int bh = blockIdx.z * KVH + blockIdx.y;
  const int n = counts[bh], per = 2 * (D / VB) + 1;
  const int2 *list = pairs + (size_t)bh * max_moves;
  const size_t row0 = (size_t)bh * T_cap;
  const long long items = (long long)n * per;
  for (long long e = (long long)blockIdx.x * kMoveThreads + threadIdx.x; e < items;
       e += (long long)gridDim.x * kMoveThreads) {
    const int m = (int)(e / per), i = (int)(e - (long long)m * per);
    const size_t to = row0 + list[m].x, from = row0 + list[m].y;
    if (i < per - 1) {
      int8_t *c = i < D / VB ? kc : vc;
      const size_t at = (size_t)(i < D / VB ? i : i - D / VB) * VB;
      if constexpr (VB == 16) *(u32x4 *)(c + to * D + at) = *(const u32x4 *)(c + from * D + at);
      else *(u32x2 *)(c + to * D + at) = *(const u32x2 *)(c + from * D + at);
    } else {
      if constexpr (SB == 2) {
        ((uint16_t *)ks)[to] = ((const uint16_t *)ks)[from];
        ((uint16_t *)vs)[to] = ((const uint16_t *)vs)[from];
      } else {
        ((uint32_t *)ks)[to] = ((const uint32_t *)ks)[from];
        ((uint32_t *)vs)[to] = ((const uint32_t *)vs)[from];
      }
      scores[to] = scores[from];
      positions[to] = positions[from];
    }
  }
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
  k_evict_select<<<dim3(KVH, B), kSelThreads, 0, st>>>(scores, positions, lengths, T, seen, seen_host, budget,
                                                      recent, lengths_out, counts, pairs, most, KVH, T_cap);
  if (most) {
    const bool wide = D % 16 == 0 && (((uintptr_t)k_codes | (uintptr_t)v_codes) & 15) == 0;
    const long long items = (long long)most * (2 * (D / (wide ? 16 : 8)) + 1);
    const long long blocks = (items + kMoveThreads - 1) / kMoveThreads;
    const dim3 grid((unsigned)(blocks < 64 ? blocks : 64), KVH, B);
#define SF_MOVE(VB, SB)                                                                                     \
  k_evict_move<VB, SB><<<grid, kMoveThreads, 0, st>>>(k_codes, k_scales, v_codes, v_scales, scores, positions, \
                                                      counts, pairs, most, KVH, T_cap, D)
    if (wide) {
      if (scale_dtype == SF_F16) SF_MOVE(16, 2);
      else SF_MOVE(16, 4);
    } else {
      if (scale_dtype == SF_F16) SF_MOVE(8, 2);
      else SF_MOVE(8, 4);
    }
#undef SF_MOVE
  }
  return sf_check_launch("sf_kv_evict");
}
