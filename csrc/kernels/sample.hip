// One class drawn from every row of logits with temperature, top-k, top-p and min-p, from given
// random numbers.
//
// With x = (z - max z) / T and w = exp(x), and a row's classes in order (larger logit first, then lower
// class), the filters keep, one after another:
//   top-k: the k first classes (k <= 0: all);
//   top-p: of those, the classes whose preceding mass in the order is below p times their mass, the
//          first always (p >= 1: all);
//   min-p: of those, the ones with w >= min_p (the largest has w = 1; min_p <= 0: all).
// The draw is the first class, in class order, whose cumulative kept mass exceeds u times the kept
// mass, u clamped into [0, 1); prob is its share of the kept mass. T <= 0 takes the first maximum; T = inf or NaN counts as the
// largest finite number.
// Masked classes (-inf, NaN) are never drawn; a row without any other gives class -1, prob 0.
//
// Masses are integer sums of fixed-point weights (logit_rows.h), so a draw does not depend on how the
// row is cut over threads. What the filters keep is a prefix of the order, given by its last class (Keep).
//
// Which kernel draws a row:
//   rows of up to 2048 classes: one wave, from registers (sample_wave_kernel);
//   longer rows with a short top-k: the k first classes by one pass (row_top.h), few long rows in parts;
//   longer rows else: one block, from memory, a pass of weights and one of those kept (sample_row_kernel).
// Bound by the issue of the weights' f64 instructions, 26 per logit: 65536 x 1000 f32 without filters 78 to 84 us (85 %
// of it issue), p = 0.9: 181 us, k = 50: 149 us; 256 x 65537 bf16, p = 0.9: 66 to 70 us. By two launches where few rows
// have a short top-k: 1 x 131072 f32, k = 50: 16 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdexcept>
#include <type_traits>

#include "kernels/row_top.h"
#include "mlapi/common.h"
#include "mlapi/kernels.h"

namespace mlapi {
namespace {

using namespace lrow;

struct Settings {
  float T, top_p, min_p;
  int top_k;
  double c;  // log2(e) / T
};

// c_all: log2(e) / temperature_all, divided on the host (a division in 64 bits is 15 instructions)
struct Call : SampleCall {
  double c_all;
};

__device__ __forceinline__ Settings settings(const Call& a, int64_t row) {
  Settings s;
  // finite: an infinite temperature times an infinite difference, a masked class's, is no number
  s.T = fminf(a.temperature != nullptr ? a.temperature[row] : a.temperature_all, 0x1.fffffep127f);
  s.c = a.temperature != nullptr ? 1.4426950408889634074 / (double)s.T : a.c_all;
  s.top_p = a.top_p != nullptr ? a.top_p[row] : a.top_p_all;
  s.min_p = a.min_p != nullptr ? a.min_p[row] : a.min_p_all;
  s.top_k = a.top_k != nullptr ? a.top_k[row] : a.top_k_all;
  return s;
}
__device__ __forceinline__ float uniform(const Call& a, int64_t row) {
  return fminf(fmaxf(a.u[row], 0.f), 0x1.fffffep-1f);  // NaN: 0
}
// the smallest weight that min-p keeps
__device__ __forceinline__ uint64_t least_weight(float min_p) {
  if (__builtin_amdgcn_readfirstlane(min_p > 0.f ? 1 : 0) == 0) return 0;  // the same for the row
  return (uint64_t)__builtin_ceil((double)fminf(min_p, 1.f) * (double)(1ull << WEIGHT_BITS));
}

// What is left of a row after top-k and top-p: the classes up to one in the order, and a least weight.
struct Keep {
  float m;
  double c;
  float z;  // the last class kept: its logit and its number
  int cls;
  uint64_t least;
  // every class is kept
  __device__ __forceinline__ bool all() const { return z == -__builtin_inff() && least == 0; }
  __device__ __forceinline__ uint64_t any_mass(float x) const { return weight(no_nan(x), m, c); }
  __device__ __forceinline__ uint64_t mass(float x, int i) const {
    const uint64_t w = any_mass(x);
    return (x > z || (x == z && i <= cls)) && w >= least ? w : 0;
  }
  __device__ __forceinline__ void upto(uint64_t place, Places places) { places.upto(place, z, cls); }
};

__device__ __forceinline__ Keep keep_all(float m, const Settings& set) {
  return Keep{m, set.c, -__builtin_inff(), 0x7fffffff, least_weight(set.min_p)};
}

// ---- from a sorted list ---------------------------------------------------------------------------
// The draw among the first n classes of a row, sorted places in LDS, by one wave; top-k is done. `w` and
// `c` hold n entries.
template <int MAX>
__device__ __forceinline__ void draw_from_list(const Call& a, int64_t row, const Settings& set, Places places,
                               const uint64_t* sorted, int n, int lane, uint64_t* w, int* c) {
  n = __builtin_amdgcn_readfirstlane(n);
  constexpr int PER = MAX / 64;
  const Keep keep = keep_all(key_logit((uint32_t)(sorted[0] >> places.ib)), set);
  uint64_t own[PER], mass = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = i * 64 + lane;
    own[i] = 0;
    if (i * 64 < n && r < n) own[i] = weight(key_logit((uint32_t)(sorted[r] >> places.ib)), keep.m, keep.c);
    mass += own[i];
  }
  const uint64_t target = set.top_p < 1.f ? ceil_part(wave_sum_int(mass), fmaxf(set.top_p, 0.f)) : ~(uint64_t)0;
  uint64_t before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (i * 64 >= n) continue;
    const int r = i * 64 + lane;
    const uint64_t upto = before + wave_scan(own[i], lane);
    before = lane_value(upto, 63);
    const bool in = r == 0 || upto - own[i] < target;
    own[i] = in && own[i] >= keep.least ? own[i] : 0;
    total += own[i];
    if (r < n) w[r] = own[i], c[r] = places.cls(sorted[r]);
  }
  total = wave_sum_int(total);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const uint64_t t = floor_part(total, uniform(a, row));
  auto pick = [&](auto rounds) {
    constexpr int R = decltype(rounds)::value;
    int mine[R];
    uint64_t lower[R];  // the kept mass of lower classes
#pragma unroll
    for (int i = 0; i < R; ++i) mine[i] = i * 64 + lane < n ? c[i * 64 + lane] : -1, lower[i] = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const uint64_t wj = w[j];
      const int cj = c[j];
#pragma unroll
      for (int i = 0; i < R; ++i) lower[i] += cj < mine[i] ? wj : 0;
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (own[i] != 0 && lower[i] <= t && t < lower[i] + own[i]) {
        a.idx[row] = mine[i];
        a.prob[row] = (float)((double)own[i] / (double)total);
      }
  };
  if (n <= 64)
    pick(std::integral_constant<int, 1>{});
  else
    pick(std::integral_constant<int, PER>{});
}

__device__ __forceinline__ void write_one(const Call& a, int64_t row, int cls, float prob) {
  a.idx[row] = cls;
  a.prob[row] = prob;
}

// ---- one wave, row in registers -------------------------------------------------------------------
constexpr int WAVE_BINS = 256;
constexpr int WAVE_LIST = 256;
constexpr int WAVE_SHORT = 64;  // longest top-k by a list: 64 rows of 1000, k = 50: 9 us (20 at 128), by a cut 16 at any k
struct WaveLds {
  union {
    struct {
      WaveTopLds top;
      uint64_t w[WAVE_SHORT];
      int c[WAVE_SHORT];
    } l;
    struct {
      uint64_t mass[WAVE_BINS], place[WAVE_LIST], w[WAVE_LIST];
    } h;
    SelectLds<WAVE_BINS> select;
  } u;
};

// ALL: the call has neither top-k nor top-p. Up to 16 classes per lane fit four waves on a SIMD; three, of 131
// registers, took 209 us for 65536 rows of 1000 at p = 0.9, four 178.
template <class T, int NV, bool ALL>
__global__ __launch_bounds__(256, NV * Vec<T>::N <= 16 ? 4 : 2) void sample_wave_kernel(Call a) {
  constexpr int V = Vec<T>::N;
  __shared__ WaveLds lds[ALL ? 1 : 4];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= a.B) return;
  const int K = a.K;
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  Held<T> raw[NV];
  load_row<T, 64, NV>(raw, z, lane, K);
  const Settings set = settings(a, row);
  float m = -__builtin_inff();
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < V; ++e) m = fmaxf(m, raw[v][e]);
  m = wave_max(m);
  auto pass = [&](auto f) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const Held<T> h = raw[v].fresh();
#pragma unroll
      for (int e = 0; e < V; ++e) f(h[e], (v * 64 + lane) * V + e);
    }
  };
  if (m == -__builtin_inff() || !(set.T > 0.f)) {
    int first = K;
    pass([&](float x, int i) { first = x == m ? min(first, i) : first; });
    first = wave_reduce(first, [](int x, int y) { return min(x, y); });
    const bool none = m == -__builtin_inff();
    if (lane == 0) write_one(a, row, none ? -1 : first, none ? 0.f : 1.f);
    return;
  }
  Keep keep = keep_all(m, set);
  if constexpr (!ALL) {
    WaveLds& s = lds[wave];
    const Places places(K);
    if (set.top_k > 0 && set.top_k <= WAVE_SHORT) {
      const int n = wave_top<T, NV>(raw, lane, K, set.top_k, &s.u.l.top);
      draw_from_list<WAVE_SHORT>(a, row, set, places, s.u.l.top.sorted, n, lane, s.u.l.w, s.u.l.c);
      return;
    }
    // every weight once; a class that a filter drops loses its weight
    uint64_t w[NV * V];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < V; ++e) w[v * V + e] = keep.any_mass(raw[v][e]);
    auto each = [&](auto f) {  // f(class, logit, weight)
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int e = 0; e < V; ++e) f((v * 64 + lane) * V + e, raw[v][e], w[v * V + e]);
    };
    auto by_place = [&](auto f) {
      each([&](int i, float x, uint64_t wi) {
        const uint32_t key = order_key(x);
        if (key > KEY_MASKED) f(places.of(key, i), wi);
      });
    };
    auto drop = [&] {  // what lies past the last class kept
      each([&](int i, float x, uint64_t& wi) { wi = x > keep.z || (x == keep.z && i <= keep.cls) ? wi : 0; });
    };
    const uint64_t lo = places.last(KEY_MASKED + 1), hi = places.first(order_key(m)) - 1;
    if (set.top_k > 0 && set.top_k < K) {
      wave_cut<T, NV>(raw, lane, K, set.top_k, keep.z, keep.cls);
      drop();
    }
    if (set.top_p < 1.f) {
      uint64_t mass = 0;
      each([&](int, float, uint64_t wi) { mass += wi; });
      const uint64_t part = ceil_part(wave_sum_int(mass), fmaxf(set.top_p, 0.f)), target = part == 0 ? 1 : part;
      // masses by bins of equal width in z, as for a long row (below)
      constexpr int PER = WAVE_BINS / 64;
#pragma unroll
      for (int b = 0; b < PER; ++b) s.u.h.mass[b * 64 + lane] = 0;
      const float scale = (float)(WAVE_BINS / 30.0) / set.T;
      auto depth = [&](float x) { return fminf(fmaxf((m - x) * scale, 0.f), (float)(WAVE_BINS - 1)); };
      auto sync = [] {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      };
      sync();
      each([&](int, float x, uint64_t wi) {
        if (wi != 0) atomicAdd((unsigned long long*)&s.u.h.mass[(int)depth(x)], (unsigned long long)wi);
      });
      sync();
      uint64_t bin[PER], own = 0;
#pragma unroll
      for (int b = 0; b < PER; ++b) own += bin[b] = s.u.h.mass[lane * PER + b];
      const uint64_t upto = wave_scan(own, lane);
      uint64_t before = upto - own;
      int at = 0;
      const uint64_t hit = __ballot(before < target && upto >= target);
#pragma unroll
      for (int b = 0; b < PER - 1; ++b)
        if (before + bin[b] < target && at == b) before += bin[b], ++at;
      const int where = __builtin_ctzll(hit);
      const uint64_t above = lane_value(before, where);
      const float near = (float)lane_value(lane * PER + at, where);
      int n = 0;
      each([&](int i, float x, uint64_t wi) {
        const float d = depth(x);
        const bool in = wi != 0 && d >= near && d < near + 1.f;
        const uint64_t mk = __ballot(in);
        if (mk != 0) {
          const int j = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(mk >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mk, 0));
          if (in && j < WAVE_LIST) s.u.h.place[j] = places.of(order_key(x), i), s.u.h.w[j] = wi;
          n += __popcll(mk);
        }
      });
      sync();
      if (n <= WAVE_LIST) {
        uint64_t last = 0;
        for (int j0 = 0; j0 < n; j0 += 64) {
          const int j = j0 + lane;
          const uint64_t mine = j < n ? s.u.h.place[j] : 0, wj = j < n ? s.u.h.w[j] : 0;
          uint64_t sum = above;
#pragma unroll 4
          for (int i = 0; i < n; ++i) sum += s.u.h.place[i] > mine ? s.u.h.w[i] : 0;
          const uint64_t hits = __ballot(j < n && sum < target && sum + wj >= target);
          if (hits != 0) last = lane_value(mine, __builtin_ctzll(hits));
        }
        keep.upto(last, places);
      } else {
        keep.upto(select_prefix<64, WAVE_BINS>(true, target, lo, hi, &s.u.select, by_place).cut, places);
      }
      drop();
    }
    each([&](int, float, uint64_t& wi) { wi = wi >= keep.least ? wi : 0; });
    uint64_t by_vec[NV], total = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      by_vec[v] = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) by_vec[v] += w[v * V + e];
      total += by_vec[v];
    }
    total = wave_sum_int(total);
    const uint64_t t = floor_part(total, uniform(a, row));
    uint64_t base = 0;  // the kept mass of the vectors before v
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const uint64_t upto = base + wave_scan(by_vec[v], lane);
      uint64_t before = upto - by_vec[v];
      base = lane_value(upto, 63);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint64_t wi = w[v * V + e];
        if (t >= before && t < before + wi)
          write_one(a, row, (v * 64 + lane) * V + e, (float)((double)wi / (double)total));
        before += wi;
      }
    }
    return;
  }
  // without filters: the kept mass vector by vector, then within the drawn one
  uint64_t w[NV * V], by_vec[NV], total = 0;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    by_vec[v] = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) by_vec[v] += w[v * V + e] = keep.any_mass(raw[v][e]);
  }
  if (keep.least != 0) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      by_vec[v] = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) by_vec[v] += w[v * V + e] = w[v * V + e] >= keep.least ? w[v * V + e] : 0;
    }
  }
  uint64_t upto[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    upto[v] = total + wave_scan(by_vec[v], lane);
    total = lane_value(upto[v], 63);
  }
  const uint64_t t = floor_part(total, uniform(a, row));
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    uint64_t before = upto[v] - by_vec[v];
    if (t >= before && t < upto[v]) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint64_t wi = w[v * V + e];
        if (t >= before && t < before + wi)
          write_one(a, row, (v * 64 + lane) * V + e, (float)((double)wi / (double)total));
        before += wi;
      }
    }
  }
}

// ---- long rows with a short top-k -----------------------------------------------------------------
struct ListLds {
  BlockTopLds top;
  uint64_t w[BLOCK_TOP];
  int c[BLOCK_TOP];
};

__device__ __forceinline__ bool short_list(const Settings& set) { return set.top_k > 0 && set.top_k <= BLOCK_TOP; }

__device__ __forceinline__ void draw_or_none(const Call& a, int64_t row, Settings set, Places places, int n,
                                             ListLds* s) {
  if (threadIdx.x >= 64) return;
  if (n == 0) {
    if (threadIdx.x == 0) write_one(a, row, -1, 0.f);
  } else if (!(set.T > 0.f)) {
    if (threadIdx.x == 0) write_one(a, row, places.cls(s->top.sorted[0]), 1.f);
  } else {
    draw_from_list<BLOCK_TOP>(a, row, set, places, s->top.sorted, n, threadIdx.x, s->w, s->c);
  }
}

// rows whose top-k is not short are left to another kernel
template <class T>
__global__ __launch_bounds__(TOP_THREADS) void sample_list_kernel(Call a) {
  __shared__ ListLds s;
  const int64_t row = blockIdx.x;
  const Settings set = settings(a, row);
  if (!short_list(set)) return;
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  const Places places(a.K);
  const int n = block_top<T>(z, 0, a.K, places, set.top_k, &s.top);
  draw_or_none(a, row, set, places, n, &s);
}

// lists[row][part][k], k the same for all rows
template <class T>
__global__ __launch_bounds__(TOP_THREADS) void sample_parts_kernel(Call a, int len, uint64_t* lists) {
  __shared__ BlockTopLds s;
  const int64_t row = blockIdx.y;
  const int k = a.top_k_all, c0 = blockIdx.x * len;
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  const int n = block_top<T>(z, c0, min(a.K, c0 + len), Places(a.K), k, &s);
  uint64_t* out = lists + (row * gridDim.x + blockIdx.x) * k;
  for (int r = threadIdx.x; r < k; r += TOP_THREADS) out[r] = r < n ? s.sorted[r] : 0;
}
__global__ __launch_bounds__(TOP_THREADS) void sample_merge_kernel(Call a, int parts, const uint64_t* lists) {
  __shared__ ListLds s;
  const int64_t row = blockIdx.x;
  const int k = a.top_k_all;
  const Places places(a.K);
  const int n = merge_top(lists + row * parts * k, parts * k, places, k, &s.top);
  draw_or_none(a, row, settings(a, row), places, n, &s);
}

// ---- one block, row in memory ---------------------------------------------------------------------
// A row is read four times: for its maximum, the masses by logit, the classes next to the border, the
// masses by class. The reads after the first come from the caches and cost little beside the weights:
// 256 rows of 65536 bf16 took 68 us with the row in registers, whose unrolled passes outgrow the
// instruction cache.
constexpr int MASS_LIST = 1024;
template <class T, int NT>
struct RowLds {
  // twice the threads: 65536 normal logits leave about 150 classes in the bin of a border
  static constexpr int BINS = NT < 512 ? 1024 : 2 * NT;
  static constexpr int SEGMENTS = NT < 512 ? 1024 : LOGIT_MAX_CLASSES / 256;  // a wave's vectors of one step
  union {
    struct {
      uint64_t mass[BINS];
      uint64_t place[MASS_LIST], w[MASS_LIST];
    } h;
    uint64_t segment[SEGMENTS];
    SelectLds<SELECT_BINS> select;
  } u;
  T kept[NT / 64][64 * Vec<T>::N];  // of a wave's vectors
  uint64_t scratch[NT / 64];
  uint64_t out[3];
  int n;
};
constexpr int SMALL_BLOCK_CLASSES = 8192;  // longest rows of 256 threads: 32 segments

// Where the running sum of x[0 .. NT PER) (PER to a thread, in order) passes `target(sum of all)`: out = index,
// sum before it, target. The sum of all reaches the target.
template <int NT, int PER, class Target>
__device__ __forceinline__ void crossing(const uint64_t* x, int count, uint64_t* scratch, uint64_t* out,
                                         Target&& target) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint64_t own = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (tid * PER + i < count) own += x[tid * PER + i];
  uint64_t upto = wave_scan(own, lane), all = 0;
  __syncthreads();
  if (lane == 63) scratch[wave] = upto;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wave) upto += scratch[w];
    all += scratch[w];
  }
  const uint64_t t = target(all);
  uint64_t before = upto - own;
  if (before < t && upto >= t) {
    int i = tid * PER;
    while (before + x[i] < t) before += x[i++];
    out[0] = i, out[1] = before, out[2] = t;
  }
  __syncthreads();
}

// SKIP: rows with a short top-k have been drawn already
template <class T, int NT, bool SKIP>
__global__ __launch_bounds__(NT) void sample_row_kernel(Call a) {
  constexpr int V = Vec<T>::N, STEP = NT * V, WAVES = NT / 64, U = 2;
  typedef RowLds<T, NT> Lds;
  __shared__ Lds s;
  const int64_t row = blockIdx.x;
  const Settings set = settings(a, row);
  if (SKIP && short_list(set)) return;
  const int K = a.K, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  const Places places(K);
  // one pass over the row: f(vector, its first class), for every thread the same number of times
  auto vectors = [&](auto f) {
    int base = 0;
    for (; base + U * STEP <= K; base += U * STEP) {
      Held<T> h[U];
#pragma unroll
      for (int u = 0; u < U; ++u) h[u].load(z, base + u * STEP + tid * V);
#pragma unroll
      for (int u = 0; u < U; ++u) f(h[u], base + u * STEP + tid * V);
    }
    for (; base < K; base += STEP) {
      Held<T> h;
      h.load(z, base + tid * V, K);
      f(h, base + tid * V);
    }
  };
  auto pass = [&](auto f) {
    vectors([&](const Held<T>& h, int i) {
#pragma unroll
      for (int e = 0; e < V; ++e) f(h[e], i + e);
    });
  };
  float m = -__builtin_inff();
  pass([&](float x, int) { m = fmaxf(m, x); });
  const float largest = m;  // this thread's
  m = block_reduce<NT>(m, reinterpret_cast<float*>(s.scratch), [](float x, float y) { return fmaxf(x, y); });
  if (m == -__builtin_inff() || !(set.T > 0.f)) {
    int first = K;
    pass([&](float x, int i) { first = x == m && i < K ? min(first, i) : first; });
    first = block_reduce<NT>(first, reinterpret_cast<int*>(s.scratch), [](int x, int y) { return min(x, y); });
    const bool none = m == -__builtin_inff();
    if (tid == 0) write_one(a, row, none ? -1 : first, none ? 0.f : 1.f);
    return;
  }
  Keep keep = keep_all(m, set);
  auto each = [&](auto f) {
    pass([&](float x, int i) {
      const uint32_t key = order_key(x);
      if (key > KEY_MASKED) f(places.of(key, i), weight(x, m, keep.c));
    });
  };
  uint64_t lo = places.last(KEY_MASKED + 1);
  const uint64_t hi = places.first(order_key(m)) - 1;
  if (set.top_k > 0 && set.top_k < K) {
    int valid = 0;
    pass([&](float x, int) { valid += x > -__builtin_inff() ? 1 : 0; });
    valid = block_reduce<NT>(valid, reinterpret_cast<int*>(s.scratch), [](int x, int y) { return x + y; });
    if (set.top_k < valid) {
      auto places_only = [&](auto f) {
        pass([&](float x, int i) {
          const uint32_t key = order_key(x);
          if (key > KEY_MASKED) f(places.of(key, i), (uint64_t)0);
        });
      };
      const uint32_t bound = key_bound<NT>(order_key(largest), set.top_k, s.u.select.count);
      if (bound > KEY_MASKED) lo = places.last(bound);
      lo = select_prefix<NT, SELECT_BINS>(false, set.top_k, lo, hi, &s.u.select, places_only).cut;
      keep.upto(lo, places);
      __syncthreads();
    }
  }
  if (set.top_p < 1.f) {
    // masses by bins of equal width in z, the largest logit in bin 0; past 30 T a weight is nothing
    for (int b = tid; b < Lds::BINS; b += NT) s.u.h.mass[b] = 0;
    if (tid == 0) s.n = 0;
    __syncthreads();
    const float scale = (float)(Lds::BINS / 30.0) / set.T;
    auto depth = [&](float x) { return fminf(fmaxf((m - x) * scale, 0.f), (float)(Lds::BINS - 1)); };
    const Keep first{m, keep.c, keep.z, keep.cls, 0};
    auto count = [&](float x, uint64_t w) {
      if (w != 0) atomicAdd((unsigned long long*)&s.u.h.mass[(int)depth(x)], (unsigned long long)w);
    };
    if (first.all())
      pass([&](float x, int) { count(x, first.any_mass(x)); });
    else
      pass([&](float x, int i) { count(x, first.mass(x, i)); });
    __syncthreads();
    crossing<NT, Lds::BINS / NT>(s.u.h.mass, Lds::BINS, s.scratch, s.out, [&](uint64_t mass) {
      const uint64_t t = ceil_part(mass, fmaxf(set.top_p, 0.f));
      return t == 0 ? 1 : t;
    });
    const uint64_t above = s.out[1], target = s.out[2];
    const float near = (float)(int)s.out[0];
    // the classes of that bin, still kept by top-k; their weights once they are few
    const uint64_t from = lo;
    pass([&](float x, int i) {
      const float d = depth(x);
      if (d >= near && d < near + 1.f) {
        const uint32_t key = order_key(x);
        const uint64_t place = places.of(key, i);
        if (key > KEY_MASKED && place >= from) {
          const int j = atomicAdd(&s.n, 1);
          if (j < MASS_LIST) s.u.h.place[j] = place;
        }
      }
    });
    __syncthreads();
    const int n = s.n;
    if (n <= MASS_LIST) {
      for (int j = tid; j < n; j += NT)
        s.u.h.w[j] = weight(key_logit((uint32_t)(s.u.h.place[j] >> places.ib)), m, keep.c);
      __syncthreads();
      for (int j = tid; j < n; j += NT) {
        const uint64_t mine = s.u.h.place[j], w = s.u.h.w[j];
        uint64_t before = above;
#pragma unroll 4
        for (int i = 0; i < n; ++i) before += s.u.h.place[i] > mine ? s.u.h.w[i] : 0;
        if (before < target && before + w >= target) s.out[0] = mine;
      }
      __syncthreads();
      lo = s.out[0];
    } else {  // many classes next to the border: equal logits, or a wide bin
      lo = select_prefix<NT, SELECT_BINS>(true, target, lo, hi, &s.u.select, each).cut;
    }
    keep.upto(lo, places);
    __syncthreads();
  }
  // kept mass of every wave's vectors of one step, in class order
  auto segments = [&](auto mass) {
    vectors([&](const Held<T>& h, int i) {
      uint64_t w = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) w += mass(h[e], i + e);
      w = wave_sum_int(w);
      if (lane == 0) s.u.segment[i / (64 * V)] = w;
    });
  };
  if (keep.z == -__builtin_inff()) {
    segments([&](float x, int) {
      const uint64_t w = keep.any_mass(x);
      return w >= keep.least ? w : 0;
    });
  } else {
    // The classes kept of a vector, close together: a weight costs more than finding it a lane (256 x 65536
    // bf16, p = 0.9, 1 class in 4 kept: 62 us, 70 with a weight for every class; with nearly all kept 78 and 75).
    T* mine = s.kept[wave];
    vectors([&](const Held<T>& h, int i) {
      int n = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x = h[e];
        const uint64_t in = __ballot(x > keep.z || (x == keep.z && i + e <= keep.cls));
        const int at =
            n + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
        if (in >> lane & 1) mine[at] = (T)x;
        n += __popcll(in);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      uint64_t w = 0;
      for (int j = 0; j < n; j += 64) {
        const uint64_t wj = j + lane < n ? weight((float)mine[j + lane], m, keep.c) : 0;
        w += wj >= keep.least ? wj : 0;
      }
      w = wave_sum_int(w);
      if (lane == 0) s.u.segment[i / (64 * V)] = w;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    });
  }
  __syncthreads();
  uint64_t total = 0;
  const int count = (K + STEP - 1) / STEP * WAVES;
  crossing<NT, Lds::SEGMENTS / NT>(s.u.segment, count, s.scratch, s.out, [&](uint64_t mass) {
    total = mass;
    return floor_part(mass, uniform(a, row)) + 1;  // the first sum above it
  });
  const int pick = (int)s.out[0];
  if (wave != pick % WAVES) return;
  const uint64_t t = s.out[2] - 1 - s.out[1];
  Held<T> h;
  const int i = pick * 64 * V + lane * V;
  h.load(z, i, K);
  uint64_t own[V], sum = 0;
#pragma unroll
  for (int e = 0; e < V; ++e) sum += own[e] = keep.mass(h[e], i + e);
  uint64_t before = wave_scan(sum, lane) - sum;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if (t >= before && t < before + own[e]) write_one(a, row, i + e, (float)((double)own[e] / (double)total));
    before += own[e];
  }
}

struct Plan {
  int parts = 1, len = 0;
};

// As top_logits cuts rows, where one short k holds for all of them.
template <class T>
Plan make_plan(const SampleCall& a) {
  Plan p;
  p.len = a.K;
  if (a.top_k != nullptr || a.top_k_all < 1 || a.top_k_all > THREAD_BOUND) return p;
  constexpr int STEP = TOP_THREADS * Vec<T>::N;
  const int steps = (a.K + STEP - 1) / STEP;
  const int64_t want = std::min<int64_t>({(512 + a.B - 1) / a.B, steps / 8, MERGE_PLACES / a.top_k_all, 64});
  p.parts = (int)std::max<int64_t>(1, want);
  p.len = (steps + p.parts - 1) / p.parts * STEP;
  p.parts = (a.K + p.len - 1) / p.len;
  return p;
}

template <class T>
bool fits_wave(int K) {
  return K <= 2048;
}

template <class T, int NV>
void launch_wave(const Call& a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.B + 3) / 4));
  const bool all = a.top_k == nullptr && a.top_k_all == 0 && a.top_p == nullptr && a.top_p_all >= 1.f;
  if (all)
    hipLaunchKernelGGL((sample_wave_kernel<T, NV, true>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((sample_wave_kernel<T, NV, false>), grid, dim3(256), 0, stream, a);
}

template <class T, bool SKIP>
void launch_row(const Call& a, hipStream_t stream) {
  const dim3 grid((unsigned)a.B);
  if (a.K <= SMALL_BLOCK_CLASSES)
    hipLaunchKernelGGL((sample_row_kernel<T, 256, SKIP>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((sample_row_kernel<T, 1024, SKIP>), grid, dim3(1024), 0, stream, a);
}

template <class T>
void run_sample(const Call& a, hipStream_t stream) {
  if (fits_wave<T>(a.K)) {
    const int vecs = (a.K + Vec<T>::N - 1) / Vec<T>::N;
    if (vecs <= 64)
      launch_wave<T, 1>(a, stream);
    else if (vecs <= 128)
      launch_wave<T, 2>(a, stream);
    else if (vecs <= 256)
      launch_wave<T, 4>(a, stream);
    else if constexpr (sizeof(T) == 4)
      launch_wave<T, 8>(a, stream);
  } else if (a.top_k != nullptr) {  // each row its own k: the short ones first, the others after
    hipLaunchKernelGGL((sample_list_kernel<T>), dim3((unsigned)a.B), dim3(TOP_THREADS), 0, stream, a);
    launch_row<T, true>(a, stream);
  } else if (a.top_k_all >= 1 && a.top_k_all <= BLOCK_TOP) {
    const Plan p = make_plan<T>(a);
    if (p.parts == 1) {
      hipLaunchKernelGGL((sample_list_kernel<T>), dim3((unsigned)a.B), dim3(TOP_THREADS), 0, stream, a);
    } else {
      uint64_t* lists = static_cast<uint64_t*>(a.workspace);
      hipLaunchKernelGGL((sample_parts_kernel<T>), dim3((unsigned)p.parts, (unsigned)a.B), dim3(TOP_THREADS), 0, stream,
                         a, p.len, lists);
      hipLaunchKernelGGL(sample_merge_kernel, dim3((unsigned)a.B), dim3(TOP_THREADS), 0, stream, a, p.parts, lists);
    }
  } else {
    launch_row<T, false>(a, stream);
  }
  MLAPI_HIP_CHECK(hipGetLastError());
}

template <class T>
size_t list_bytes(const SampleCall& a) {
  if (fits_wave<T>(a.K)) return 0;
  const Plan p = make_plan<T>(a);
  return p.parts == 1 ? 0 : (size_t)a.B * p.parts * a.top_k_all * sizeof(uint64_t);
}

}  // namespace

size_t sample_workspace(const SampleCall& c) {
  if (c.B <= 0 || c.K < 1) return 0;
  return c.dt == DT_F32 ? list_bytes<float>(c) : list_bytes<__bf16>(c);
}

void launch_sample(const SampleCall& c, hipStream_t stream) {
  if (c.B <= 0) return;
  if (c.K < 1 || c.K > LOGIT_MAX_CLASSES) throw std::invalid_argument("sample: 1 <= K <= 2^20 classes");
  if (c.ldz < c.K) throw std::invalid_argument("sample: row stride below K");
  if (c.B > 0x7fffffff) throw std::invalid_argument("sample: more than 2^31 rows");
  if (c.ws_bytes < sample_workspace(c)) throw std::invalid_argument("sample: workspace too small");
  if (c.dt != DT_F32 && c.dt != DT_BF16 && c.dt != DT_F16)
    throw std::invalid_argument("sample: logits f32, bf16 or f16");
  const int64_t step = logit_slice_rows(c.B);
  for (int64_t r0 = 0; r0 < c.B; r0 += step) {
    Call a;
    static_cast<SampleCall&>(a) = c;
    a.c_all = 1.4426950408889634074 / (double)std::min(c.temperature_all, 0x1.fffffep127f);
    a.B = std::min(step, c.B - r0);
    a.Z = static_cast<const char*>(c.Z) + r0 * c.ldz * (int64_t)dtype_size(c.dt);
    a.u = c.u + r0, a.idx = c.idx + r0, a.prob = c.prob + r0;
    if (c.temperature != nullptr) a.temperature = c.temperature + r0;
    if (c.top_k != nullptr) a.top_k = c.top_k + r0;
    if (c.top_p != nullptr) a.top_p = c.top_p + r0;
    if (c.min_p != nullptr) a.min_p = c.min_p + r0;
    if (c.dt == DT_F32)
      run_sample<float>(a, stream);
    else if (c.dt == DT_BF16)
      run_sample<__bf16>(a, stream);
    else
      run_sample<_Float16>(a, stream);
  }
}

}  // namespace mlapi
