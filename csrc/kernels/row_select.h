// Selection in the order of a row's classes by one block: the shortest prefix of the order whose
// count (or mass of fixed-point weights) reaches a target, by histograms in LDS.
#pragma once
#include "kernels/logit_rows.h"

namespace mlapi {
namespace lrow {

// A class's place in the order as one number: the logit's key above, the class counted down below.
// Larger is earlier, no two classes share one.
struct Places {
  int ib;  // bits of a class
  __host__ __device__ explicit Places(int K) : ib(K <= 1 ? 1 : 32 - __builtin_clz((unsigned)(K - 1))) {}
  __host__ __device__ __forceinline__ uint64_t of(uint32_t key, int i) const {
    return ((uint64_t)key << ib) | (uint64_t)((1u << ib) - 1u - (unsigned)i);
  }
  __device__ __forceinline__ uint64_t first(uint32_t key) const { return ((uint64_t)key + 1) << ib; }  // exclusive
  __device__ __forceinline__ uint64_t last(uint32_t key) const { return (uint64_t)key << ib; }
  __host__ __device__ __forceinline__ int cls(uint64_t place) const {
    return (int)((1u << ib) - 1u - (unsigned)(place & ((1u << ib) - 1u)));
  }
  // The classes from a place upwards, told without their keys: those with x > z, or x == z and a class of at
  // most `last`. A border that a search found may have a key that no logit has: past KEY_BELOW_ZERO, whose
  // float equals the zeros above it, every zero is.
  __host__ __device__ __forceinline__ void upto(uint64_t place, float& z, int& last) const {
    const uint32_t key = (uint32_t)(place >> ib);
    z = key_logit(key);
    last = key == KEY_BELOW_ZERO ? 0x7fffffff : cls(place);
  }
};

// the largest value that at least k of the wave's 64 M values reach (0 if none is): bit by bit, counted by
// ballots, from `top` downwards. Stops early where exactly k values are left.
template <int M, class U>
__device__ __forceinline__ U kth_largest(const U (&v)[M], int k, int bits) {
  U t = 0;
  for (int b = bits - 1; b >= 0; --b) {
    const U cand = t | ((U)1 << b);
    int n = 0;
#pragma unroll
    for (int i = 0; i < M; ++i) n += __popcll(__ballot(v[i] >= cand));
    if (n >= k) t = cand;
    if (n == k) break;
  }
  return t;
}

// A key that at least k classes of a row reach (0: fewer than k threads have a class): the k-th largest of
// the largest keys of NT threads. `lds` holds NT values. What lies below needs no bin of select_prefix,
// whose first round would else count most of a row in the few bins its exponents fall into.
template <int NT>
__device__ __forceinline__ uint32_t key_bound(uint32_t own, int k, uint32_t* lds) {
  __syncthreads();
  lds[threadIdx.x] = own > KEY_MASKED ? own : 0;
  __syncthreads();
  uint32_t v[NT / 64];
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) v[i] = lds[i * 64 + (threadIdx.x & 63)];
  const uint32_t t = kth_largest<NT / 64, uint32_t>(v, k, 32);
  __syncthreads();
  return t;
}

struct Prefix {
  uint64_t cut;    // places >= cut are in it
  uint64_t count;  // classes in it
  uint64_t mass;   // their weights (0 where the count was the target)
};

constexpr int SELECT_BINS = 1024;
template <int BINS>
struct SelectLds {
  uint64_t mass[BINS];
  uint32_t count[BINS];
  uint64_t out[4];
};

// each(f): calls f(place, weight) for every class of this thread with a weight or count to give; all
// threads of the block together cover the row. target >= 1 and reached by the whole row. The interval
// of places that holds the target's class is cut into BINS bins until one class (or an exact end) is
// left: 1024 bins take one or two rounds for logits without many ties. A wave of its own (NT 64) needs no
// barrier of its block.
template <int NT, int BINS, class Each>
__device__ __forceinline__ Prefix select_prefix(const bool by_mass, uint64_t target, uint64_t lo, uint64_t hi,
                                                SelectLds<BINS>* s, Each&& each) {
  constexpr int PER = BINS / 64, LOG = __builtin_ctz(BINS);
  const int tid = NT == 64 ? (int)threadIdx.x & 63 : (int)threadIdx.x;
  auto sync = [] {
    if constexpr (NT == 64) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    } else {
      __syncthreads();
    }
  };
  uint64_t above_n = 0, above_m = 0;
  for (;;) {
    const uint64_t range = hi - lo;
    const int bits = range == 0 ? 0 : 64 - __builtin_clzll(range);
    const int sh = bits > LOG ? bits - LOG : 0;
    sync();
    for (int b = tid; b < BINS; b += NT) s->mass[b] = 0, s->count[b] = 0;
    sync();
    each([&](uint64_t place, uint64_t w) {
      if (place >= lo && place <= hi) {
        const int b = (int)((place - lo) >> sh);
        atomicAdd(&s->count[b], 1u);
        if (by_mass) atomicAdd((unsigned long long*)&s->mass[b], (unsigned long long)w);
      }
    });
    sync();
    if (tid < 64) {
      // lane l: bins [PER l, PER l + PER); the lanes above come first in the order
      const int l = tid;
      uint64_t n = 0, m = 0;
      for (int b = 0; b < PER; ++b) n += s->count[l * PER + b], m += s->mass[l * PER + b];
      const uint64_t tn = wave_sum_int(n), tm = wave_sum_int(m);
      const uint64_t pn = above_n + tn - wave_scan(n, l), pm = above_m + tm - wave_scan(m, l);  // before this lane's
      const uint64_t before = by_mass ? pm : pn, own = by_mass ? m : n;
      if (before < target && before + own >= target) {
        uint64_t cn = pn, cm = pm;
        for (int b = l * PER + PER - 1;; --b) {
          const uint64_t nn = cn + s->count[b], nm = cm + s->mass[b];
          if ((by_mass ? nm : nn) >= target || b == l * PER) {
            s->out[0] = b, s->out[1] = cn, s->out[2] = cm;
            break;
          }
          cn = nn, cm = nm;
        }
      }
    }
    sync();
    const int b = (int)s->out[0];
    above_n = s->out[1], above_m = s->out[2];
    const uint64_t n = s->count[b], m = s->mass[b];
    lo += (uint64_t)b << sh;
    if (sh == 0 || n == 1 || (by_mass ? above_m + m : above_n + n) == target) {
      sync();
      return Prefix{lo, above_n + n, above_m + m};
    }
    const uint64_t top = lo + (((uint64_t)1 << sh) - 1);
    hi = top < hi ? top : hi;
  }
}

}  // namespace lrow
}  // namespace mlapi
