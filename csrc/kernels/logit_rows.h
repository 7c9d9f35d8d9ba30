// Device helpers of the row operators over class logits (top_logits.hip, distill.hip, sample.hip):
// 16-byte row loads at any alignment, reductions over the threads that share a row, the total order
// of a row's classes, and fixed-point weights.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace mlapi {
namespace lrow {

// A row is read 16 bytes per lane. Rows of an odd stride start at any element: the type's own
// alignment is all that is promised, and gfx950 loads and stores 16 bytes from there.
template <class T>
struct Vec {
  static constexpr int N = 16 / (int)sizeof(T);
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

template <class T>
__device__ __forceinline__ T minus_inf() {
  return (T)(-__builtin_inff());
}

// element i of a row whose address is the same for the wave: 32-bit offsets from a scalar base (64-bit
// ones cost two registers for every vector of a row)
template <class T>
__device__ __forceinline__ T* elem(T* row, int i) {
  return reinterpret_cast<T*>(reinterpret_cast<char*>(row) + (size_t)((uint32_t)i * (uint32_t)sizeof(T)));
}
template <class T>
__device__ __forceinline__ const T* elem(const T* row, int i) {
  return reinterpret_cast<const T*>(reinterpret_cast<const char*>(row) + (size_t)((uint32_t)i * (uint32_t)sizeof(T)));
}

// elements [i, i + N) of a row of K; those past its end read as -inf (a masked class) and are not loaded
template <class T>
__device__ __forceinline__ typename Vec<T>::type load_vec(const T* row, int i, int K) {
  constexpr int N = Vec<T>::N;
  if (i + N <= K) return *reinterpret_cast<const typename Vec<T>::type*>(elem(row, i));
  typename Vec<T>::type v;
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = i + e < K ? *elem(row, i + e) : minus_inf<T>();
  return v;
}

// A vector held over several passes of a row in registers. Each pass unpacks it anew (refresh): left
// alone, the compiler keeps the f32 values of 16-bit types from the first pass, twice the registers.
template <class T>
struct Held {
  typedef uint32_t raw_t __attribute__((ext_vector_type(4)));
  raw_t raw;
  __device__ __forceinline__ void load(const T* row, int i) {
    raw = __builtin_bit_cast(raw_t, *reinterpret_cast<const typename Vec<T>::type*>(elem(row, i)));
  }
  __device__ __forceinline__ void load(const T* row, int i, int K) {
    raw = __builtin_bit_cast(raw_t, load_vec(row, i, K));
  }
  __device__ __forceinline__ void mask() { raw = __builtin_bit_cast(raw_t, masked()); }
  __device__ __forceinline__ void refresh() { asm volatile("" : "+v"(raw)); }
  // a copy for one pass, where a refresh in place would stand under a condition (and leave a second
  // copy of the whole row for the other branch)
  __device__ __forceinline__ Held fresh() const {
    Held h = *this;
    h.refresh();
    return h;
  }
  __device__ __forceinline__ float operator[](int e) const {
    typedef T vec_t __attribute__((ext_vector_type(Vec<T>::N)));
    return (float)__builtin_bit_cast(vec_t, raw)[e];
  }
  static __device__ __forceinline__ auto masked() {
    typedef T vec_t __attribute__((ext_vector_type(Vec<T>::N)));
    return (vec_t)(minus_inf<T>());
  }
};

// A row's NV vectors per thread, NTR threads: vector v of thread t holds classes [(v NTR + t) N, + N), -inf
// past the row's end. Only one step of NTR vectors can be cut by that end: its guarded loads come once.
template <class T, int NTR, int NV>
__device__ __forceinline__ void load_row(Held<T> (&raw)[NV], const T* row, int tid, int K) {
  constexpr int STEP = NTR * Vec<T>::N;
  const int whole = K / STEP;  // the same for the wave
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (v < whole)
      raw[v].load(row, v * STEP + tid * Vec<T>::N);
    else
      raw[v].mask();
  }
  if (whole < NV && whole * STEP < K) {
    Held<T> last;
    last.load(row, whole * STEP + tid * Vec<T>::N, K);
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (v == whole) raw[v] = last;
  }
}

// ---- reductions over a wave: DPP within its rows of 16 lanes, then through scalar registers ---------
// (a shuffle through LDS costs its latency at each of six steps). The tree is always the same.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {  // lanes without a source read 0
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(uint32_t, v)));
}
template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
  return (int)dpp<CTRL>((uint32_t)v);
}
template <int CTRL>
__device__ __forceinline__ uint64_t dpp(uint64_t v) {
  return (uint64_t)dpp<CTRL>((uint32_t)(v >> 32)) << 32 | dpp<CTRL>((uint32_t)v);
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); }
__device__ __forceinline__ int lane_value(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
__device__ __forceinline__ float lane_value(float v, int l) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
}
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int l) {
  return (uint64_t)lane_value((uint32_t)(v >> 32), l) << 32 | lane_value((uint32_t)v, l);
}
constexpr int ROW_ROR = 0x120, ROW_SHR = 0x110;
// op over the 16 lanes of a row, to all of them
template <class U, class Op>
__device__ __forceinline__ U row_reduce(U v, Op op) {
  v = op(v, dpp<ROW_ROR + 8>(v));
  v = op(v, dpp<ROW_ROR + 4>(v));
  v = op(v, dpp<ROW_ROR + 2>(v));
  return op(v, dpp<ROW_ROR + 1>(v));
}
template <class U, class Op>
__device__ __forceinline__ U wave_reduce(U v, Op op) {
  v = row_reduce(v, op);
  return op(op(lane_value(v, 0), lane_value(v, 16)), op(lane_value(v, 32), lane_value(v, 48)));
}
__device__ __forceinline__ float wave_max(float v) {
  return wave_reduce(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_reduce(v, [](float x, float y) { return x + y; });
}
template <class U>
__device__ __forceinline__ U wave_sum_int(U v) {
  return wave_reduce(v, [](U x, U y) { return x + y; });
}
// inclusive prefix sum over the lanes
template <class U>
__device__ __forceinline__ U wave_scan(U v, int lane) {
  v += dpp<ROW_SHR + 1>(v);
  v += dpp<ROW_SHR + 2>(v);
  v += dpp<ROW_SHR + 4>(v);
  v += dpp<ROW_SHR + 8>(v);
  const U a = lane_value(v, 15), b = lane_value(v, 31), c = lane_value(v, 47);
  return v + (lane >= 48 ? a + b + c : lane >= 32 ? a + b : lane >= 16 ? a : 0);
}

// Over a block of NT threads; `scratch` holds NT / 64 values and may be used again after the call.
template <int NT, class U, class Op>
__device__ __forceinline__ U block_reduce(U v, U* scratch, Op op) {
  v = wave_reduce(v, op);
  if constexpr (NT > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    v = scratch[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v = op(v, scratch[w]);
    __syncthreads();
  }
  return v;
}

// ---- the order of a row's classes: larger logit first, then lower class -------------------------
// An unsigned key that rises with the logit: -0 as +0; NaN as -inf. Masked classes (-inf, NaN) have
// KEY_MASKED, every other key is larger. No logit has KEY_BELOW_ZERO, whose float is -0.
constexpr uint32_t KEY_MASKED = 0x007fffffu, KEY_BELOW_ZERO = 0x7fffffffu;
__host__ __device__ __forceinline__ uint32_t order_key(float z) {
  const uint32_t b = __builtin_bit_cast(uint32_t, z + 0.0f);
  const uint32_t key = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return z != z ? KEY_MASKED : key;
}
__host__ __device__ __forceinline__ float key_logit(uint32_t key) {
  const uint32_t b = key ^ ((key & 0x80000000u) ? 0x80000000u : 0xffffffffu);
  return __builtin_bit_cast(float, b);
}

// ---- fixed-point weights ------------------------------------------------------------------------
// w(z) = 2^42 exp((z - m) / T), rounded, m the row's maximum. Integer sums of these do not depend on
// their order, so masses found by atomics, by lanes or by blocks agree to the bit, and 2^20 of them
// stay below 2^63. The step of 2^-42 of the largest weight is what a border between two classes can
// be off by: the exponential is evaluated in f64 (an f32 one, 2^-24 off, would move a border of 65536
// rows of 1000 classes often enough to be seen).
constexpr int WEIGHT_BITS = 42;
// z may be -inf (weight 0) but not NaN.
__device__ __forceinline__ uint64_t weight(float z, float m, double c /* log2(e) / T */) {
  // from above: inf - inf, a NaN, where m is inf; from below: all that rounds to nothing
  const double x = __builtin_fma((double)z - (double)m, c, (double)WEIGHT_BITS);
  const double y = __builtin_fmax(__builtin_fmin(x, (double)WEIGHT_BITS), -16.0);
  const double n = __builtin_rint(y), f = y - n;
  // 2^f on [-1/2, 1/2]: 1 + f q(f), q of degree 8 through (2^f - 1) / f at nine Chebyshev points,
  // 2^-44.6 off; exactly 1 at f = 0, so equal logits weigh the same
  double p = 0x1.b638718fee5a8p-24;
  p = __builtin_fma(p, f, 0x1.63d136366db24p-20);
  p = __builtin_fma(p, f, 0x1.ffcb95269d85ap-17);
  p = __builtin_fma(p, f, 0x1.4308ac85aa947p-13);
  p = __builtin_fma(p, f, 0x1.5d87fe86f82cdp-10);
  p = __builtin_fma(p, f, 0x1.3b2ab7181b755p-7);
  p = __builtin_fma(p, f, 0x1.c6b08d7047e8bp-5);
  p = __builtin_fma(p, f, 0x1.ebfbdff823cedp-3);
  p = __builtin_fma(p, f, 0x1.62e42fefa39efp-1);
  p = __builtin_fma(p, f, 1.0);
  // the integer nearest to p 2^n falls out of the low bits of a sum with 2^52
  const double w = __builtin_ldexp(p, (int)n) + 0x1p52;
  return __builtin_bit_cast(uint64_t, w) & 0xfffffffffffffull;
}
__device__ __forceinline__ float no_nan(float z) { return fmaxf(z, -__builtin_inff()); }

// floor(u mass) and ceil(p mass) for a fraction 0 <= u, p < 1, exactly
__device__ __forceinline__ uint64_t fraction_bits(float u) { return (uint64_t)((double)u * 0x1p64); }
__device__ __forceinline__ uint64_t floor_part(uint64_t mass, float u) { return __umul64hi(mass, fraction_bits(u)); }
__device__ __forceinline__ uint64_t ceil_part(uint64_t mass, float p) {
  const uint64_t f = fraction_bits(p);
  return __umul64hi(mass, f) + (mass * f != 0 ? 1 : 0);
}

}  // namespace lrow
}  // namespace mlapi
