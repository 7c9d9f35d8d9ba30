// The k first classes of every row of logits, in order: larger logit first, then lower class.
//
// A row's k-th place is found by cutting the interval of places into bins until exactly k classes lie
// above a bound (row_select.h); the k classes found are ranked by counting the larger ones.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdexcept>

#include "kernels/row_select.h"
#include "mlapi/common.h"
#include "mlapi/kernels.h"

namespace mlapi {
namespace {

using namespace lrow;

struct TopArgs {
  const void* Z;
  void* values;
  int32_t* idx;
  int64_t B, ldz;
  int K, k;
};

template <class T, int NT>
__global__ __launch_bounds__(NT) void top_block_kernel(TopArgs a) {
  constexpr int V = Vec<T>::N;
  __shared__ SelectLds sel;
  __shared__ uint64_t list[LOGIT_MAX_TOP];
  __shared__ uint32_t scratch[NT / 64];
  __shared__ int found;
  const int64_t row = blockIdx.x;
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  const Places places(a.K);
  uint32_t hi = 0, lo = 0xffffffffu, n = 0;
  for (int i = (int)threadIdx.x * V; i < a.K; i += NT * V) {
    const typename Vec<T>::type raw = load_vec(z, i, a.K);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const uint32_t key = order_key((float)raw[e]);
      if (key > KEY_MASKED) hi = max(hi, key), lo = min(lo, key), ++n;
    }
  }
  hi = block_reduce<NT>(hi, scratch, [](uint32_t x, uint32_t y) { return max(x, y); });
  lo = block_reduce<NT>(lo, scratch, [](uint32_t x, uint32_t y) { return min(x, y); });
  n = block_reduce<NT>(n, scratch, [](uint32_t x, uint32_t y) { return x + y; });
  const int take = (int)min(n, (uint32_t)a.k);
  T* values = static_cast<T*>(a.values) + row * a.k;
  int32_t* idx = a.idx + row * a.k;
  for (int r = take + threadIdx.x; r < a.k; r += NT) values[r] = minus_inf<T>(), idx[r] = -1;
  if (take == 0) return;
  auto each = [&](auto f) {
    for (int i = (int)threadIdx.x * V; i < a.K; i += NT * V) {
      const typename Vec<T>::type raw = load_vec(z, i, a.K);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t key = order_key((float)raw[e]);
        if (key > KEY_MASKED) f(places.of(key, i + e), (uint64_t)0);
      }
    }
  };
  const Prefix p = select_prefix<NT>(false, take, places.last(lo), places.first(hi) - 1, &sel, each);
  if (threadIdx.x == 0) found = 0;
  __syncthreads();
  each([&](uint64_t place, uint64_t) {
    if (place >= p.cut) list[atomicAdd(&found, 1)] = place;
  });
  __syncthreads();
  for (int j = threadIdx.x; j < take; j += NT) {
    const uint64_t mine = list[j];
    int r = 0;
    for (int i = 0; i < take; ++i) r += list[i] > mine ? 1 : 0;
    const int c = places.cls(mine);
    values[r] = z[c];
    idx[r] = c;
  }
}

template <class T>
void run_top(const TopArgs& a, hipStream_t stream) {
  if (a.K <= 8192) {
    hipLaunchKernelGGL((top_block_kernel<T, 256>), dim3((unsigned)a.B), dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL((top_block_kernel<T, 1024>), dim3((unsigned)a.B), dim3(1024), 0, stream, a);
  }
  MLAPI_HIP_CHECK(hipGetLastError());
}

}  // namespace

size_t top_logits_workspace(int dt, int64_t B, int K, int k) {
  (void)dt, (void)B, (void)K, (void)k;
  return 0;
}

void launch_top_logits(int dt, const void* Z, int64_t ldz, int64_t B, int K, int k, void* values, int32_t* idx,
                       void* workspace, size_t ws_bytes, hipStream_t stream) {
  (void)workspace, (void)ws_bytes;
  if (B <= 0) return;
  if (K < 1 || K > LOGIT_MAX_CLASSES || k < 1 || k > LOGIT_MAX_TOP)
    throw std::invalid_argument("top_logits: 1 <= K <= 2^20 classes, 1 <= k <= 1024");
  if (ldz < K) throw std::invalid_argument("top_logits: row stride below K");
  if (B > 0x7fffffff) throw std::invalid_argument("top_logits: more than 2^31 rows");
  const TopArgs a{Z, values, idx, B, ldz, K, k};
  if (dt == DT_F32) return run_top<float>(a, stream);
  if (dt == DT_BF16) return run_top<__bf16>(a, stream);
  if (dt == DT_F16) return run_top<_Float16>(a, stream);
  throw std::invalid_argument("top_logits: logits f32, bf16 or f16");
}

}  // namespace mlapi
