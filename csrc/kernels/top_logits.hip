// The k first classes of every row of logits, in order: larger logit first, then lower class.
//
// Bound by reading the logits once: one comparison per logit, and work on about k classes after it
// (row_top.h). Short rows stay in one wave's registers, no barrier; a long row takes a block; a few long
// rows are cut into parts whose sorted lists a second launch merges. Lists too long for those
// (k > 256) are found by cutting the interval of places into bins (row_select.h).
// 65536 x 1000 f32, k = 16: 60 us, 4.5 TB/s; 1023 x 131072 bf16, k = 64: 62 us, 4.4 TB/s (k = 256: 111); 512 x 40000
// f32, k = 400: 73 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <stdexcept>

#include "kernels/row_top.h"
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

template <class T>
__device__ __forceinline__ void write_top(const TopArgs& a, int64_t row, const T* z, Places places,
                                          const uint64_t* sorted, int n, int tid, int threads) {
  T* values = static_cast<T*>(a.values) + row * a.k;
  int32_t* idx = a.idx + row * a.k;
  for (int r = tid; r < a.k; r += threads) {
    const int c = r < n ? places.cls(sorted[r]) : -1;
    values[r] = r < n ? z[c] : minus_inf<T>();  // the logit itself: its key has lost the sign of a zero
    idx[r] = c;
  }
}

template <class T, int NV>
__global__ __launch_bounds__(256) void top_wave_kernel(TopArgs a) {
  __shared__ WaveTopLds lds[4];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= a.B) return;
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  Held<T> raw[NV];
  load_row<T, 64, NV>(raw, z, lane, a.K);
  const int n = wave_top<T, NV>(raw, lane, a.K, a.k, &lds[wave]);
  write_top<T>(a, row, z, Places(a.K), lds[wave].sorted, n, lane, 64);
}

template <class T>
__global__ __launch_bounds__(TOP_THREADS) void top_row_kernel(TopArgs a) {
  __shared__ BlockTopLds lds;
  const int64_t row = blockIdx.x;
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  const int n = block_top<T>(z, 0, a.K, Places(a.K), a.k, &lds);
  write_top<T>(a, row, z, Places(a.K), lds.sorted, n, threadIdx.x, TOP_THREADS);
}

// lists[row][part][k]: the sorted places of a part, 0 past them
template <class T>
__global__ __launch_bounds__(TOP_THREADS) void top_parts_kernel(TopArgs a, int len, uint64_t* lists) {
  __shared__ BlockTopLds lds;
  const int64_t row = blockIdx.y;
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  const int c0 = blockIdx.x * len;
  const int n = block_top<T>(z, c0, min(a.K, c0 + len), Places(a.K), a.k, &lds);
  uint64_t* out = lists + (row * gridDim.x + blockIdx.x) * a.k;
  for (int r = threadIdx.x; r < a.k; r += TOP_THREADS) out[r] = r < n ? lds.sorted[r] : 0;
}

template <class T>
__global__ __launch_bounds__(TOP_THREADS) void top_merge_kernel(TopArgs a, int parts, const uint64_t* lists) {
  __shared__ BlockTopLds lds;
  const int64_t row = blockIdx.x;
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  const int n = merge_top(lists + row * parts * a.k, parts * a.k, Places(a.K), a.k, &lds);
  write_top<T>(a, row, z, Places(a.K), lds.sorted, n, threadIdx.x, TOP_THREADS);
}

template <class T, int NT>
__global__ __launch_bounds__(NT) void top_select_kernel(TopArgs a) {
  constexpr int V = Vec<T>::N;
  __shared__ SelectLds<SELECT_BINS> sel;
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
  const uint32_t own = hi;  // this thread's largest
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
  lo = max(lo, key_bound<NT>(own, take, sel.count));
  const Prefix p = select_prefix<NT, SELECT_BINS>(false, take, places.last(lo), places.first(hi) - 1, &sel, each);
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

struct Plan {
  int parts = 1, len = 0;
};

// A row is cut where there are fewer rows than 512 blocks (two on each CU), into parts of at least
// 8 steps, with lists that the merge holds.
template <class T>
Plan make_plan(int64_t B, int K, int k) {
  Plan p;
  constexpr int STEP = TOP_THREADS * Vec<T>::N;
  p.len = K;
  if (k > THREAD_BOUND) return p;  // the merge bounds lists by its threads
  const int steps = (K + STEP - 1) / STEP;
  const int64_t want = std::min<int64_t>({(512 + B - 1) / B, steps / 8, MERGE_PLACES / k, 64});
  p.parts = (int)std::max<int64_t>(1, want);
  p.len = (steps + p.parts - 1) / p.parts * STEP;
  p.parts = (K + p.len - 1) / p.len;
  return p;
}

template <class T, int NV>
void launch_wave(const TopArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((top_wave_kernel<T, NV>), dim3((unsigned)((a.B + 3) / 4)), dim3(256), 0, stream, a);
  MLAPI_HIP_CHECK(hipGetLastError());
}

template <class T>
bool fits_wave(int K, int k) {
  return k <= WAVE_TOP && K <= 64 * 8 * Vec<T>::N;
}

template <class T>
void run_top(const TopArgs& a, uint64_t* lists, hipStream_t stream) {
  const int vecs = (a.K + Vec<T>::N - 1) / Vec<T>::N;
  if (fits_wave<T>(a.K, a.k)) {
    if (vecs <= 64) return launch_wave<T, 1>(a, stream);
    if (vecs <= 128) return launch_wave<T, 2>(a, stream);
    if (vecs <= 256) return launch_wave<T, 4>(a, stream);
    return launch_wave<T, 8>(a, stream);
  }
  if (a.k <= BLOCK_TOP) {
    const Plan p = make_plan<T>(a.B, a.K, a.k);
    if (p.parts == 1) {
      hipLaunchKernelGGL((top_row_kernel<T>), dim3((unsigned)a.B), dim3(TOP_THREADS), 0, stream, a);
    } else {  // few rows: they fit grid.y
      hipLaunchKernelGGL((top_parts_kernel<T>), dim3((unsigned)p.parts, (unsigned)a.B), dim3(TOP_THREADS), 0, stream, a,
                         p.len, lists);
      hipLaunchKernelGGL((top_merge_kernel<T>), dim3((unsigned)a.B), dim3(TOP_THREADS), 0, stream, a, p.parts, lists);
    }
  } else if (a.K <= 8192) {
    hipLaunchKernelGGL((top_select_kernel<T, 256>), dim3((unsigned)a.B), dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL((top_select_kernel<T, 1024>), dim3((unsigned)a.B), dim3(1024), 0, stream, a);
  }
  MLAPI_HIP_CHECK(hipGetLastError());
}

template <class T>
size_t list_bytes(int64_t B, int K, int k) {
  if (fits_wave<T>(K, k) || k > BLOCK_TOP) return 0;
  const Plan p = make_plan<T>(B, K, k);
  return p.parts == 1 ? 0 : (size_t)B * p.parts * k * sizeof(uint64_t);
}

}  // namespace

size_t top_logits_workspace(int dt, int64_t B, int K, int k) {
  if (B <= 0 || K < 1 || k < 1) return 0;
  return dt == DT_F32 ? list_bytes<float>(B, K, k) : list_bytes<__bf16>(B, K, k);
}

void launch_top_logits(int dt, const void* Z, int64_t ldz, int64_t B, int K, int k, void* values, int32_t* idx,
                       void* workspace, size_t ws_bytes, hipStream_t stream) {
  if (B <= 0) return;
  if (K < 1 || K > LOGIT_MAX_CLASSES || k < 1 || k > LOGIT_MAX_TOP)
    throw std::invalid_argument("top_logits: 1 <= K <= 2^20 classes, 1 <= k <= 1024");
  if (ldz < K) throw std::invalid_argument("top_logits: row stride below K");
  if (B > 0x7fffffff) throw std::invalid_argument("top_logits: more than 2^31 rows");
  if (ws_bytes < top_logits_workspace(dt, B, K, k)) throw std::invalid_argument("top_logits: workspace too small");
  if (dt != DT_F32 && dt != DT_BF16 && dt != DT_F16)
    throw std::invalid_argument("top_logits: logits f32, bf16 or f16");
  uint64_t* lists = static_cast<uint64_t*>(workspace);
  const int64_t step = logit_slice_rows(B), size = (int64_t)dtype_size(dt);
  for (int64_t r0 = 0; r0 < B; r0 += step) {
    const TopArgs a{static_cast<const char*>(Z) + r0 * ldz * size, static_cast<char*>(values) + r0 * k * size, idx + r0 * k,
                    std::min(step, B - r0), ldz, K, k};
    if (dt == DT_F32)
      run_top<float>(a, lists, stream);
    else if (dt == DT_BF16)
      run_top<__bf16>(a, lists, stream);
    else
      run_top<_Float16>(a, lists, stream);
  }
}

}  // namespace mlapi
