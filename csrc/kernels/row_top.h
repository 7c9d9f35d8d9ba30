// The first k classes of a row, sorted, in LDS: by one wave from registers (short rows), by one block in
// one pass over memory (long rows), or from the lists of a row's parts.
//
// All three rest on one bound: take the largest place of every group of a partition of the row; the k-th
// largest of these is at most the row's k-th place, so no class below it is among the first k. With n
// groups about n ln(n / (n - k)) classes of a row without a pattern lie above the bound: little more
// than k for n >= 2 k. They are gathered and each is ranked by counting the larger ones. Rows whose
// pattern leaves more than fit (ties, one group holding all that is large) are cut exactly instead.
#pragma once
#include "kernels/row_select.h"

namespace mlapi {
namespace lrow {

// Ranks n distinct places in LDS (by how many are larger) over THREADS threads, each holding PER of them:
// sorted[r] gets the place of rank r < k. Every place is read once by all, four at a time: `cand` is padded
// with zeros to a multiple of four.
template <int THREADS, int PER>
__device__ __forceinline__ void rank_some(const uint64_t* cand, int n, int k, int tid, uint64_t* sorted) {
  uint64_t mine[PER];
  int rank[PER];
#pragma unroll
  for (int p = 0; p < PER; ++p) mine[p] = tid + p * THREADS < n ? cand[tid + p * THREADS] : ~(uint64_t)0, rank[p] = 0;
#pragma unroll 1
  for (int i = 0; i < n; i += 4) {
    const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(cand + i), y = *reinterpret_cast<const ulonglong2*>(cand + i + 2);
#pragma unroll
    for (int p = 0; p < PER; ++p)
      rank[p] += (x.x > mine[p] ? 1 : 0) + (x.y > mine[p] ? 1 : 0) + (y.x > mine[p] ? 1 : 0) + (y.y > mine[p] ? 1 : 0);
  }
#pragma unroll
  for (int p = 0; p < PER; ++p)
    if (tid + p * THREADS < n && rank[p] < k) sorted[rank[p]] = mine[p];
}
// n is the same for all threads
template <int THREADS, int MOST>
__device__ __forceinline__ void rank_places(const uint64_t* cand, int n, int k, int tid, uint64_t* sorted) {
  if (n <= THREADS) return rank_some<THREADS, 1>(cand, n, k, tid, sorted);
  if (n <= 2 * THREADS) return rank_some<THREADS, 2>(cand, n, k, tid, sorted);
  rank_some<THREADS, MOST>(cand, n, k, tid, sorted);
}

// ---- one wave, row in registers -----------------------------------------------------------------
constexpr int WAVE_TOP = 256;   // longest list
constexpr int WAVE_CAND = 512;  // gathered classes
struct alignas(16) WaveTopLds {
  uint64_t cand[WAVE_CAND + 4];
  uint64_t sorted[WAVE_TOP];
};

// Gathers the classes of a row in registers whose keys are above `over`, or equal to it with a class of
// at most `last`. Returns how many there are (more than WAVE_CAND: not all were written).
template <class T, int NV>
__device__ __forceinline__ int wave_gather(const Held<T> (&raw)[NV], int lane, Places places, float over, int last,
                                           uint64_t* list) {
  constexpr int V = Vec<T>::N;
  int n = 0;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float z = raw[v][e];
      const int i = (v * 64 + lane) * V + e;
      const bool in = z >= over && z > -__builtin_inff() && (z > over || i <= last);
      const uint64_t m = __ballot(in);
      if (m != 0) {
        const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
        if (in && at < WAVE_CAND) list[at] = places.of(order_key(z), i);
        n += __popcll(m);
      }
    }
  return n;
}

// Where the first k classes of a row in registers end, exactly: they are those with z > over, or z == over
// and a class of at most `last` (and not masked). The k-th largest key bit by bit, then, among the classes that
// share it, the last that fits.
template <class T, int NV>
__device__ __forceinline__ void wave_cut(const Held<T> (&raw)[NV], int lane, int K, int k, float& over, int& last) {
  constexpr int V = Vec<T>::N;
  const Places places(K);
  auto count = [&](auto pred) {
    int c = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < V; ++e) c += __popcll(__ballot(pred(raw[v][e], (v * 64 + lane) * V + e)));
    return c;
  };
  const float inf = __builtin_inff();
  over = -inf, last = K;
  if (count([&](float z, int) { return z > -inf; }) <= k) return;
  uint32_t t = 0;
#pragma unroll 1
  for (int b = 31; b >= 0; --b) {
    const float cand = key_logit(t | 1u << b);  // NaN keys: no logit reaches them
    if (count([&](float z, int) { return z >= cand; }) >= k) t |= 1u << b;
  }
  over = key_logit(t);
  const int ties = k - count([&](float z, int) { return z > over; });
  last = 0;  // the smallest class by which `ties` classes tie
#pragma unroll 1
  for (int b = places.ib - 1; b >= 0; --b) {
    const int below = last + (1 << b) - 1;
    if (count([&](float z, int i) { return z == over && i <= below; }) < ties) last += 1 << b;
  }
}

// Sorts the first k (at most WAVE_TOP) classes of the row into s->sorted; returns their number.
template <class T, int NV>
__device__ __forceinline__ int wave_top(const Held<T> (&raw)[NV], int lane, int K, int k, WaveTopLds* s) {
  constexpr int V = Vec<T>::N;
  const Places places(K);
  // groups: a lane's whole share, or each of its vectors
  float most = -__builtin_inff();
  uint32_t by_vec[NV], by_lane[1];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float x = raw[v][0];
#pragma unroll
    for (int e = 1; e < V; ++e) x = fmaxf(x, raw[v][e]);
    by_vec[v] = order_key(x);
    most = fmaxf(most, x);
  }
  by_lane[0] = order_key(most);
  uint32_t bound = KEY_MASKED;
  if (k <= 32)
    bound = kth_largest<1, uint32_t>(by_lane, k, 32);
  else if (k <= 32 * NV)
    bound = kth_largest<NV, uint32_t>(by_vec, k, 32);
  int n = WAVE_CAND + 1;
  if (bound > KEY_MASKED) n = wave_gather<T, NV>(raw, lane, places, key_logit(bound), K, s->cand);
  if (n > WAVE_CAND) {
    float over;
    int last;
    wave_cut<T, NV>(raw, lane, K, k, over, last);
    n = wave_gather<T, NV>(raw, lane, places, over, last, s->cand);
  }
  n = __builtin_amdgcn_readfirstlane(n);
  if (lane < 4) s->cand[n + lane] = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  rank_places<64, WAVE_CAND / 64>(s->cand, n, k, lane, s->sorted);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  return min(n, k);
}

// ---- one block, row in memory -------------------------------------------------------------------
constexpr int TOP_THREADS = 256;
constexpr int BLOCK_TOP = 256;    // longest list
constexpr int THREAD_BOUND = 128; // longest list bounded by the threads' best places; longer ones: by the groups'
constexpr int BLOCK_CAND = 1024;  // gathered classes
constexpr int GROUP_LANES = 16;   // a group is 16 lanes' vectors of `rounds` steps: 256 bytes each
constexpr int MAX_GROUPS = 2048;
struct alignas(16) BlockTopLds {
  uint64_t cand[BLOCK_CAND + 4];
  union {
    struct {
      float most[MAX_GROUPS];
      uint16_t group[MAX_GROUPS];
    } g;
    SelectLds<SELECT_BINS> select;
  } u;
  uint64_t sorted[BLOCK_TOP];
  uint64_t best[TOP_THREADS];
  int groups, n;
};

// ranks the s->n gathered places
__device__ __forceinline__ int block_rank(int k, BlockTopLds* s) {
  const int n = __builtin_amdgcn_readfirstlane(s->n);
  if (threadIdx.x < 4) s->cand[n + threadIdx.x] = 0;
  __syncthreads();
  rank_places<TOP_THREADS, BLOCK_CAND / TOP_THREADS>(s->cand, n, k, threadIdx.x, s->sorted);
  __syncthreads();
  return min(n, k);
}

// the k-th largest of the threads' best places (0: fewer than k threads have one)
__device__ __forceinline__ uint64_t block_bound(uint64_t best, int k, int bits, BlockTopLds* s) {
  s->best[threadIdx.x] = best;
  if (threadIdx.x == 0) s->groups = 0, s->n = 0;
  __syncthreads();
  uint64_t v[TOP_THREADS / 64];
#pragma unroll
  for (int i = 0; i < TOP_THREADS / 64; ++i) v[i] = s->best[i * 64 + (threadIdx.x & 63)];
  return kth_largest<TOP_THREADS / 64, uint64_t>(v, k, bits);
}

// Sorts the first k (at most BLOCK_TOP) of the classes [c0, c1) of a row into s->sorted, by a block of
// TOP_THREADS; returns their number. One pass reads the part, keeping the largest logit of every group of
// classes and of every thread; the groups that reach the bound (about k, 256 bytes each) are read again.
template <class T>
__device__ __forceinline__ int block_top(const T* z, int c0, int c1, Places places, int k, BlockTopLds* s) {
  constexpr int V = Vec<T>::N, STEP = TOP_THREADS * V, U = 4;
  const int tid = threadIdx.x, steps = (c1 - c0 + STEP - 1) / STEP;
  const int rounds = (steps * (TOP_THREADS / GROUP_LANES) + MAX_GROUPS - 1) / MAX_GROUPS;
  auto fmax2 = [](float x, float y) { return fmaxf(x, y); };
  float best = -__builtin_inff(), group = -__builtin_inff();
  int best_at = 0, left = rounds, g = tid / GROUP_LANES;
  for (int s0 = 0; s0 < steps; s0 += U) {
    Held<T> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int base = c0 + (s0 + u) * STEP;
      if (base + STEP <= c1)
        raw[u].load(z, base + tid * V);
      else
        raw[u].load(z, base + tid * V, c1);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x = raw[u][0];
#pragma unroll
      for (int e = 1; e < V; ++e) x = fmaxf(x, raw[u][e]);
      if (x > best) best = x, best_at = s0 + u;
      group = fmaxf(group, x);
      if (--left == 0 || s0 + u == steps - 1) {
        group = row_reduce(group, fmax2);
        if (tid % GROUP_LANES == 0 && g < MAX_GROUPS && s0 + u < steps) s->u.g.most[g] = group;
        g += TOP_THREADS / GROUP_LANES;
        group = -__builtin_inff();
        left = rounds;
      }
    }
  }
  // this thread's first class, by its first step with its largest logit (the vector's own classes share
  // one place: the bound need not be tight)
  const uint32_t key = order_key(best);
  const uint64_t mine = key > KEY_MASKED ? places.of(key, min(c0 + best_at * STEP + tid * V + V - 1, c1 - 1)) : 0;
  uint64_t bound = block_bound(mine, k, 32 + places.ib, s);
  const int ngroups = (steps + rounds - 1) / rounds * (TOP_THREADS / GROUP_LANES);
  if (k > THREAD_BOUND) {
    // 256 threads are too few groups for so many: the k-th largest of up to 2048 groups' logits, without their
    // classes (ties of that logit are gathered too)
    constexpr int PER = MAX_GROUPS / 64;
    uint32_t v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int g = i * 64 + (tid & 63);
      v[i] = g < ngroups ? order_key(s->u.g.most[g]) : 0;
    }
    const uint32_t key = kth_largest<PER, uint32_t>(v, k, 32);
    bound = key > KEY_MASKED ? places.last(key) : 0;
  }
  const float over = bound == 0 ? -__builtin_inff() : key_logit((uint32_t)(bound >> places.ib));
  for (int i = tid; i < ngroups; i += TOP_THREADS)
    if (s->u.g.most[i] >= over) s->u.g.group[atomicAdd(&s->groups, 1)] = (uint16_t)i;
  __syncthreads();
  for (int i = tid / GROUP_LANES; i < s->groups; i += TOP_THREADS / GROUP_LANES) {
    const int gi = s->u.g.group[i];
    const int first = c0 + gi / (TOP_THREADS / GROUP_LANES) * rounds * STEP +
                      (gi % (TOP_THREADS / GROUP_LANES) * GROUP_LANES + tid % GROUP_LANES) * V;
    for (int r = 0; r < rounds && first + r * STEP < c1; ++r) {
      Held<T> raw;
      raw.load(z, first + r * STEP, c1);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t kk = order_key(raw[e]);
        const uint64_t place = places.of(kk, first + r * STEP + e);
        if (kk > KEY_MASKED && place >= bound) {
          const int at = atomicAdd(&s->n, 1);
          if (at < BLOCK_CAND) s->cand[at] = place;
        }
      }
    }
  }
  __syncthreads();
  if (s->n > BLOCK_CAND) {
    auto each = [&](auto f) {
      for (int i = c0 + tid * V; i < c1; i += STEP) {
        Held<T> raw;
        raw.load(z, i, c1);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const uint32_t kk = order_key(raw[e]);
          const uint64_t place = places.of(kk, i + e);
          if (kk > KEY_MASKED && place >= bound) f(place, (uint64_t)0);
        }
      }
    };
    // more than k classes reach the bound, so the k-th place exists
    const uint64_t cut = select_prefix<TOP_THREADS, SELECT_BINS>(false, k, bound, ~(uint64_t)0 >> (32 - places.ib),
                                                    &s->u.select, each).cut;
    __syncthreads();
    if (tid == 0) s->n = 0;
    __syncthreads();
    each([&](uint64_t place, uint64_t) {
      if (place >= cut) s->cand[atomicAdd(&s->n, 1)] = place;
    });
    __syncthreads();
  }
  return block_rank(k, s);
}

// ---- from the lists of a row's parts ------------------------------------------------------------
constexpr int MERGE_PLACES = 2048;
// `lists`: count places in any order, 0 where there is none; count <= MERGE_PLACES
__device__ __forceinline__ int merge_top(const uint64_t* lists, int count, Places places, int k, BlockTopLds* s) {
  constexpr int PER = MERGE_PLACES / TOP_THREADS;
  uint64_t v[PER], best = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = i * TOP_THREADS + (int)threadIdx.x;
    v[i] = j < count ? lists[j] : 0;
    best = v[i] > best ? v[i] : best;
  }
  const uint64_t bound = block_bound(best, k, 32 + places.ib, s);
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (v[i] != 0 && v[i] >= bound) {
      const int at = atomicAdd(&s->n, 1);
      if (at < BLOCK_CAND) s->cand[at] = v[i];
    }
  __syncthreads();
  return block_rank(k, s);
}

}  // namespace lrow
}  // namespace mlapi
