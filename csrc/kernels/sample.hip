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
// mass, u clamped into [0, 1); prob is its share of the kept mass. T <= 0 (or NaN) takes the first maximum.
// Masked classes (-inf, NaN) are never drawn; a row without any other gives class -1, prob 0.
//
// Masses are integer sums of fixed-point weights (logit_rows.h), so a draw does not depend on how the
// row is cut over threads.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdexcept>

#include "kernels/row_select.h"
#include "mlapi/common.h"
#include "mlapi/kernels.h"

namespace mlapi {
namespace {

using namespace lrow;

struct Settings {
  float T, top_p, min_p;
  int top_k;
};

__device__ __forceinline__ Settings settings(const SampleCall& a, int64_t row) {
  Settings s;
  s.T = a.temperature != nullptr ? a.temperature[row] : a.temperature_all;
  s.top_p = a.top_p != nullptr ? a.top_p[row] : a.top_p_all;
  s.min_p = a.min_p != nullptr ? a.min_p[row] : a.min_p_all;
  s.top_k = a.top_k != nullptr ? a.top_k[row] : a.top_k_all;
  return s;
}
__device__ __forceinline__ float uniform(const SampleCall& a, int64_t row) {
  return fminf(fmaxf(a.u[row], 0.f), 0x1.fffffep-1f);  // NaN: 0
}
// the smallest weight that min-p keeps
__device__ __forceinline__ uint64_t least_weight(float min_p) {
  if (!(min_p > 0.f)) return 0;
  return (uint64_t)__builtin_ceil((double)fminf(min_p, 1.f) * (double)(1ull << WEIGHT_BITS));
}

template <class T, int NT>
__global__ __launch_bounds__(NT) void sample_block_kernel(SampleCall a) {
  constexpr int V = Vec<T>::N, STEP = NT * V, MAX_STEPS = NT == 1024 ? LOGIT_MAX_CLASSES / STEP : 8;
  __shared__ SelectLds sel;
  __shared__ uint64_t scratch[NT / 64];
  __shared__ uint64_t step_mass[MAX_STEPS];
  __shared__ uint64_t pick[2];
  const int64_t row = blockIdx.x;
  const int K = a.K;
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  const Places places(K);
  const Settings set = settings(a, row);
  auto add = [](uint64_t x, uint64_t y) { return x + y; };
  uint64_t best = 0;  // largest place
  uint32_t lo = 0xffffffffu, n = 0;
  for (int i = (int)threadIdx.x * V; i < K; i += STEP) {
    const typename Vec<T>::type raw = load_vec(z, i, K);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const uint32_t key = order_key((float)raw[e]);
      if (key > KEY_MASKED) {
        const uint64_t place = places.of(key, i + e);
        best = best > place ? best : place;
        lo = min(lo, key);
        ++n;
      }
    }
  }
  best = block_reduce<NT>(best, scratch, [](uint64_t x, uint64_t y) { return x > y ? x : y; });
  lo = (uint32_t)block_reduce<NT>((uint64_t)lo, scratch, [](uint64_t x, uint64_t y) { return x < y ? x : y; });
  const uint64_t valid = block_reduce<NT>((uint64_t)n, scratch, add);
  if (valid == 0 || !(set.T > 0.f)) {
    if (threadIdx.x == 0) a.idx[row] = valid == 0 ? -1 : places.cls(best), a.prob[row] = valid == 0 ? 0.f : 1.f;
    return;
  }
  const float m = key_logit((uint32_t)(best >> places.ib));
  const double c = 1.4426950408889634074 / (double)set.T;
  auto each = [&](auto f) {
    for (int i = (int)threadIdx.x * V; i < K; i += STEP) {
      const typename Vec<T>::type raw = load_vec(z, i, K);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x = (float)raw[e];
        const uint32_t key = order_key(x);
        if (key > KEY_MASKED) f(places.of(key, i + e), weight(x, m, c));
      }
    }
  };
  uint64_t cut = 0, mass = 0;
  if (set.top_k > 0 && (uint64_t)set.top_k < valid) {
    const Prefix p = select_prefix<NT>(false, (uint64_t)set.top_k, places.last(lo), best, &sel, each);
    cut = p.cut, mass = p.mass;
  } else if (set.top_p < 1.f) {
    each([&](uint64_t, uint64_t w) { mass += w; });
    mass = block_reduce<NT>(mass, scratch, add);
  }
  if (set.top_p < 1.f) {
    uint64_t target = ceil_part(mass, fmaxf(set.top_p, 0.f));
    if (target == 0) target = 1;
    const uint64_t from = cut > places.last(lo) ? cut : places.last(lo);
    cut = select_prefix<NT>(true, target, from, best, &sel, each).cut;
  }
  const uint64_t least = least_weight(set.min_p);
  // kept mass of every step of NT vectors, in class order
  const int steps = (K + STEP - 1) / STEP;
  for (int s = threadIdx.x; s < steps; s += NT) step_mass[s] = 0;
  __syncthreads();
  auto vec_mass = [&](int i) {
    uint64_t v = 0;
    if (i < K) {
      const typename Vec<T>::type raw = load_vec(z, i, K);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x = (float)raw[e];
        const uint32_t key = order_key(x);
        if (key > KEY_MASKED && places.of(key, i + e) >= cut) {
          const uint64_t w = weight(x, m, c);
          if (w >= least) v += w;
        }
      }
    }
    return v;
  };
  for (int s = 0; s < steps; ++s) {
    const uint64_t v = wave_sum_int(vec_mass(s * STEP + (int)threadIdx.x * V));
    if ((threadIdx.x & 63) == 0) atomicAdd((unsigned long long*)&step_mass[s], (unsigned long long)v);
  }
  __syncthreads();
  uint64_t total = 0;
  for (int s = 0; s < steps; ++s) total += step_mass[s];
  uint64_t t = floor_part(total, uniform(a, row));
  int s = 0;
  while (t >= step_mass[s]) t -= step_mass[s++];
  // the thread of that step, then the class of its vector
  const int i = s * STEP + (int)threadIdx.x * V;
  const uint64_t own = vec_mass(i), upto = wave_scan(own, threadIdx.x & 63);
  if ((threadIdx.x & 63) == 63) scratch[threadIdx.x >> 6] = upto;
  __syncthreads();
  uint64_t before = upto - own;
  for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) before += scratch[w];
  if (t >= before && t < before + own) {
    t -= before;
    for (int e = 0; e < V; ++e) {
      const float x = (float)z[i + e];
      const uint32_t key = order_key(x);
      if (key <= KEY_MASKED || places.of(key, i + e) < cut) continue;
      const uint64_t w = weight(x, m, c);
      if (w < least) continue;
      if (t < w) {
        a.idx[row] = i + e;
        a.prob[row] = (float)((double)w / (double)total);
        break;
      }
      t -= w;
    }
  }
}

template <class T>
void run_sample(const SampleCall& a, hipStream_t stream) {
  if (a.K <= 8 * 256 * Vec<T>::N) {
    hipLaunchKernelGGL((sample_block_kernel<T, 256>), dim3((unsigned)a.B), dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL((sample_block_kernel<T, 1024>), dim3((unsigned)a.B), dim3(1024), 0, stream, a);
  }
  MLAPI_HIP_CHECK(hipGetLastError());
}

}  // namespace

size_t sample_workspace(const SampleCall& call) {
  (void)call;
  return 0;
}

void launch_sample(const SampleCall& c, hipStream_t stream) {
  if (c.B <= 0) return;
  if (c.K < 1 || c.K > LOGIT_MAX_CLASSES) throw std::invalid_argument("sample: 1 <= K <= 2^20 classes");
  if (c.ldz < c.K) throw std::invalid_argument("sample: row stride below K");
  if (c.B > 0x7fffffff) throw std::invalid_argument("sample: more than 2^31 rows");
  if (c.dt == DT_F32) return run_sample<float>(c, stream);
  if (c.dt == DT_BF16) return run_sample<__bf16>(c, stream);
  if (c.dt == DT_F16) return run_sample<_Float16>(c, stream);
  throw std::invalid_argument("sample: logits f32, bf16 or f16");
}

}  // namespace mlapi
