// Distillation from a teacher's top logits, forward and backward, over rows of class logits.
//
// Per row of K student logits z and k teacher entries (class c_j, logit t_j), temperature T, soft share a:
//   q_j = exp(t_j / T) / sum_i exp(t_i / T)          p = softmax(z / T), p1 = softmax(z)
//   loss = a T^2 sum_j q_j (ln q_j - ln p_{c_j}) - (1 - a) ln p1_y
//   dz_i = g [ a T (p_i - sum_{j: c_j = i} q_j) + (1 - a) (p1_i - [i = y]) ]
// An entry with a negative class or a logit of -inf is absent; a row without entries (a label below 0)
// has no soft (hard) part; a row whose logits are all -inf has neither. A listed class that the student
// masks makes the loss +inf. A class of K or more, in an
// entry or a label, makes the row's loss and gradient NaN: nothing is read or written there.
//
// The gradient is dense (a softmax over K) except at the k + 1 listed classes: the row is streamed
// with the softmax alone, and the listed classes are written again afterwards with their whole value,
// computed from logits gathered before the first store (so dz may be z itself). The first entry of a
// class sums all entries of it, in their order: a class listed twice costs no atomic.
//
// Bound by memory where one softmax is asked for (a row is read once and written once, 7 operations per
// logit): 65536 x 1000 f32 with labels, loss and gradient 108 us, 4.9 TB/s; 2048 x 65536 bf16 112 us, 4.8 TB/s;
// loss and gradient apart 78 and 97 us. By the exponentials where labels at another temperature add a second softmax to
// 16-bit logits: 1501 x 32003 f16 61 us, 3.2 TB/s.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <stdexcept>

#include "kernels/logit_rows.h"
#include "mlapi/common.h"
#include "mlapi/kernels.h"

namespace mlapi {
namespace {

using namespace lrow;

// What a row's softmax needs: the maximum, sum exp((z - m) / T), sum exp(z - m), first class of the maximum.
struct RowStats {
  float m, st, s1;
  int arg;
};

__device__ __forceinline__ float finite_max(float m) { return m == -__builtin_inff() ? 0.f : m; }

struct Args {
  const void* Z;
  const int32_t* idx;
  const void* t;
  const int32_t* y;
  const float* g;
  const RowStats* stats_in;  // [B], or [B][parts] partial ones
  float* loss;
  RowStats* stats_out;
  void* dz;
  int32_t* pred;
  int32_t* near;  // [B] or null: whether a row takes 64 bits (below)
  int64_t B, ldz, ldi, ldt, ldd;
  int K, k, parts, t_dt;
  bool find;  // near is written by this launch, else read
  float T, soft, hard;  // soft = a, hard = 1 - a (0 without labels)
  bool two;             // labels at a temperature other than the teacher's: a second softmax
};

// The listed classes of one row, in LDS: n = k entries, and the label as one more; 14 bytes each, so
// that four rows of 1024 entries (and 512 bytes of bits each) stay below 64 KB.
struct Listed {
  int* cls;        // class, -1: absent
  float* x;        // (t_j - max t) log2(e) / T; q_j = 2^x_j / S
  float* z;        // its logit; later the whole gradient of the class
  uint16_t* keep;  // whether this entry writes it
  uint32_t* seen;  // a bit for every class (modulo their number): which have been listed
  __device__ Listed(unsigned char* lds, int cap) {
    cls = reinterpret_cast<int*>(lds);
    x = reinterpret_cast<float*>(cls + cap);
    z = x + cap;
    keep = reinterpret_cast<uint16_t*>(z + cap);
    seen = reinterpret_cast<uint32_t*>(keep + cap);
  }
  static __host__ __device__ int capacity(int k) { return (k + 1 + 7) / 8 * 8; }
  // 16 k^2 bits at most: two of k classes of a longer row share a bit by chance in 3 rows of 100, and
  // the walk that then looks for the class twice costs time alone
  static __host__ __device__ int bits(int k, int K) {
    int n = 256;
    while (n < K && n < 65536 && n < 16 * (k + 1) * (k + 1)) n *= 2;
    return n;
  }
  static __host__ __device__ size_t bytes(int k, int K) { return (size_t)capacity(k) * 14 + bits(k, K) / 8; }
};

// Logit j of the teacher's list of a row.
__device__ __forceinline__ float teacher_logit(const Args& a, int64_t row, int j) {
  const int64_t at = row * a.ldt + j;
  if (a.t_dt == DT_F32) return static_cast<const float*>(a.t)[at];
  if (a.t_dt == DT_BF16) return (float)static_cast<const __bf16*>(a.t)[at];
  return (float)static_cast<const _Float16*>(a.t)[at];
}

// Reads the row's entries (one wave): x (-inf: absent) and logits into z. Returns S (0 without entries), Q (1, or 0
// without entries; NaN for a class out of range or a teacher's NaN or inf), the label's weight (0 without one), and
// whether a class may stand twice among the entries.
template <class T>
__device__ __forceinline__ bool read_listed(const Args& a, int64_t row, int lane, Listed L, float& S, float& Q, float& H) {
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  const int32_t* idx = a.idx + row * a.ldi;
  const float ct = 1.44269504088896340736f / a.T;
  float mt = -__builtin_inff();
  int bad = 0, twice = 0;
  const int bits = Listed::bits(a.k, a.K);
  for (int i = lane; i < bits / 32; i += 64) L.seen[i] = 0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  auto see = [&](int c) {
    const uint32_t b = 1u << (c & 31);
    if (atomicOr(&L.seen[(c & (bits - 1)) >> 5], b) & b) twice = 1;
  };
  // four at a time: their loads wait for each other only at the gather
  for (int j0 = lane; j0 < a.k; j0 += 256) {
    int c[4];
    float x[4], zc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + 64 * i;
      c[i] = j < a.k ? idx[j] : -1;
      x[i] = j < a.k ? teacher_logit(a, row, j) : -__builtin_inff();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (c[i] < 0 || x[i] == -__builtin_inff()) c[i] = -1;
      if (c[i] >= a.K) bad = 1, c[i] = -1;
      zc[i] = c[i] < 0 ? 0.f : (float)z[c[i]];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + 64 * i;
      if (j < a.k) L.cls[j] = c[i], L.x[j] = x[i], L.z[j] = zc[i];
      if (c[i] >= 0) {
        mt = fmaxf(mt, x[i]);
        see(c[i]);
      }
    }
  }
  mt = finite_max(wave_max(mt));
  S = 0.f;
  for (int j = lane; j < a.k; j += 64) {
    // a logit near the type's lowest has no q but a finite logarithm of it: -inf times 0 is no number
    float x = (L.x[j] - mt) * ct;
    x = L.cls[j] < 0 ? -__builtin_inff() : x < -1e30f ? -1e30f : x;
    L.x[j] = x;
    S += __builtin_amdgcn_exp2f(x);
  }
  S = wave_sum(S);
  Q = S == 0.f ? 0.f : S / S;
  H = 0.f;
  int c = -1;
  if (a.hard != 0.f) {
    c = a.y[row];
    if (c >= a.K) bad = 1, c = -1;
    H = c < 0 ? 0.f : a.hard;
  }
  if (lane == 0) {
    L.cls[a.k] = c;
    L.z[a.k] = c < 0 ? 0.f : (float)z[c];
    for (int j = a.k + 1; j < Listed::capacity(a.k); ++j) L.cls[j] = -1;
  }
  if (__any(bad)) Q = __builtin_nanf("");
  return __any(twice);
}

// The row's loss (one wave; every lane gets it). S, Q and H as read_listed gave them.
__device__ float row_loss(const Args& a, int lane, Listed L, float S, float Q, float H, RowStats r) {
  if (r.st == 0.f) return Q != Q ? Q : 0.f;  // no class at all
  const float m = finite_max(r.m);
  float soft = 0.f;
  if (a.soft != 0.f && S != 0.f) {
    // T times every term, so that no finite logit overflows in a quotient by T; the sums' logarithm of their ratio: both
    // are near ln K at a high T, and what either is off counts T^2 times; a q below the type's range as 2^64 q, so
    // that it still counts against a logit near the type's lowest value; the factor of a term, not of their sum,
    // which may pass the largest number where the loss does not
    const float ratio = a.T * __logf(r.st / S), ln2_T = a.T * 0.693147180559945309f, scale = a.soft * a.T / S;
    for (int j = lane; j < a.k; j += 64) {
      if (L.cls[j] < 0) continue;
      const float term = L.x[j] * ln2_T - ((L.z[j] - m) - ratio);
      const bool low = L.x[j] < -64.f;
      const float q = __builtin_amdgcn_exp2f(low ? L.x[j] + 64.f : L.x[j]) * scale;
      soft += L.z[j] == -__builtin_inff() ? __builtin_inff() : (low ? term * 0x1p-64f : term) * q;
    }
    soft = wave_sum(soft);
  }
  float loss = soft;
  if (H != 0.f) loss += H * (__logf(r.s1) - (L.z[a.k] - m));
  return loss + (Q - Q) + (r.st - r.st);
}

// Whether p and q are near each other throughout (one wave, L as read_listed gave it): all but 1/64 of p lies on the
// listed classes. Otherwise the loss is at least T^2 / 64 of its soft part, and sums 2^-22 off show as 2^-16 of it.
__device__ bool near_rows(const Args& a, int lane, Listed L, float S, RowStats r) {
  if (a.soft == 0.f || S == 0.f || r.st == 0.f) return false;
  const float ct = 1.44269504088896340736f / a.T, m = finite_max(r.m);
  float on = 0.f;
  for (int j = lane; j < a.k; j += 64)
    if (L.cls[j] >= 0) on += __builtin_amdgcn_exp2f((L.z[j] - m) * ct);
  return wave_sum(on) > r.st * (63.f / 64.f);
}

// Coefficients of the dense part: dz_i = at exp((z_i - m) / T) + a1 exp(z_i - m).
__device__ __forceinline__ void dense_coeffs(const Args& a, float g, float Q, float H, RowStats r, float& at,
                                             float& a1) {
  const bool none = r.st == 0.f;
  at = none ? (Q - Q) : g * a.soft * a.T * Q / r.st;
  a1 = none || H == 0.f ? 0.f : g * H / r.s1;
}

// Whole gradients of the listed classes in [c0, c1), in the place of their logits; entries whose class
// another entry writes, or that lie outside, are not kept. One wave. Only a list in which a class may
// stand twice is walked for every entry (1501 x 32003 f16, k = 100: 27 us more).
__device__ __forceinline__ void listed_grads(const Args& a, int lane, Listed L, bool twice, float g, float at, float a1,
                                             float m, float S, float H, bool none, int c0, int c1) {
  const float ct = 1.44269504088896340736f / a.T, c1e = 1.44269504088896340736f;
  const float scale = S == 0.f ? 0.f : a.soft * a.T / S;
  const int cap = Listed::capacity(a.k), label = L.cls[a.k];
  auto whole = [&](int j, float sum) {
    const float d = L.z[j] - m;
    float v = none ? at : at * __builtin_amdgcn_exp2f(d * ct) - g * sum;
    if (!none && H != 0.f) v += a1 * __builtin_amdgcn_exp2f(d * c1e);
    return v;
  };
  if (!twice) {  // the label, though, is often among the entries: one of them takes its weight along
    bool listed = false;
    for (int j = lane; j < a.k; j += 64) {
      const int c = L.cls[j];
      const bool mine = c >= c0 && c < c1, both = c >= 0 && c == label;
      listed |= both;
      L.keep[j] = mine ? 1 : 0;
      if (mine) L.z[j] = whole(j, scale * __builtin_amdgcn_exp2f(L.x[j]) + (both ? H : 0.f));
    }
    listed = __any(listed);
    if (lane == 0) {
      const bool mine = label >= c0 && label < c1 && !listed;
      L.keep[a.k] = mine ? 1 : 0;
      if (mine) L.z[a.k] = whole(a.k, H);
    }
    return;
  }
  for (int j = lane; j <= a.k; j += 64) {
    const int c = L.cls[j];
    bool mine = c >= c0 && c < c1;
    float v = 0.f;
    if (mine) {
      float sum = 0.f;
      for (int i = 0; i < cap; i += 4) {
        const int4 o = *reinterpret_cast<const int4*>(L.cls + i);
        const int oc[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (oc[e] == c) {
            if (i + e < j) mine = false;
            sum += i + e == a.k ? H : scale * __builtin_amdgcn_exp2f(L.x[i + e]);
          }
      }
      v = whole(j, sum);
    }
    L.z[j] = v;
    L.keep[j] = mine ? 1 : 0;
  }
}

// ---- rows that stay in registers ----------------------------------------------------------------
// NTR threads share a row and hold NV vectors each of it; one read, one write.
template <class T, class TO, int NTR, int NV>
__global__ __launch_bounds__(NTR < 256 ? 256 : NTR, NV > 8 ? 4 : 8) void distill_rows_kernel(Args a) {
  constexpr int V = Vec<T>::N, NT = NTR < 256 ? 256 : NTR, RPB = NT / NTR;
  __shared__ float scratch[NT / 64];
  __shared__ float bcast[RPB][3];
  extern __shared__ __attribute__((aligned(16))) unsigned char dyn[];
  const int sub = RPB == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / NTR);
  const int tid = RPB == 1 ? (int)threadIdx.x : (int)threadIdx.x % NTR, lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * RPB + sub;
  if (row >= a.B) return;  // whole waves: rows of fewer than a block's threads have one wave, and no barrier
  const int K = a.K, cap = Listed::capacity(a.k);
  Listed L(dyn + (size_t)sub * Listed::bytes(a.k, a.K), cap);
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  Held<T> raw[NV];
  load_row<T, NTR, NV>(raw, z, tid, K);
  float S = 0.f, Q = 0.f, H = 0.f;
  bool twice = false;
  if (tid < 64) {
    twice = read_listed<T>(a, row, lane, L, S, Q, H);
    if (NTR > 64 && lane == 0) bcast[sub][0] = Q, bcast[sub][1] = H;
  }
  auto sync = [] {
    if constexpr (NTR > 64) {
      __syncthreads();
    } else {
      // one wave: its memory operations stay in their order, nothing to wait for
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  };
  auto again = [&] {
    if constexpr (sizeof(T) == 2 || NV >= 8) {
#pragma unroll
      for (int v = 0; v < NV; ++v) raw[v].refresh();
    }
  };
  auto fmax2 = [](float x, float y) { return fmaxf(x, y); };
  auto add2 = [](float x, float y) { return x + y; };
  const float ct = 1.44269504088896340736f / a.T, c1 = 1.44269504088896340736f;
  // The passes over the row. The refreshes stand outside of every condition: inside, each would leave a
  // second copy of the row for the other branch.
  const bool given = a.stats_in != nullptr;
  RowStats r{0.f, 0.f, 0.f, 0};
  if (given) {
    r = a.stats_in[row];
  } else {
    r.m = -__builtin_inff();
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < V; ++e) r.m = fmaxf(r.m, raw[v][e]);
    r.m = block_reduce<NTR>(r.m, scratch, fmax2);
  }
  const float m = finite_max(r.m);
  again();
  if (!given) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < V; ++e) r.st += __builtin_amdgcn_exp2f((raw[v][e] - m) * ct);
    r.st = block_reduce<NTR>(r.st, scratch, add2);
  }
  again();
  if (!given) r.s1 = a.hard != 0.f ? r.st : 0.f;
  if (!given && a.two) {
    r.s1 = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < V; ++e) r.s1 += __builtin_amdgcn_exp2f((raw[v][e] - m) * c1);
    r.s1 = block_reduce<NTR>(r.s1, scratch, add2);
  }
  again();
  if (!given && a.pred != nullptr) {
    int arg = K;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (raw[v][e] == r.m) arg = min(arg, (v * NTR + tid) * V + e);
    arg = block_reduce<NTR>(arg, reinterpret_cast<int*>(scratch), [](int x, int y) { return min(x, y); });
    r.arg = arg == K ? 0 : arg;
  }
  bool near = false;
  if (a.near != nullptr && tid < 64) {
    near = near_rows(a, lane, L, S, r);
    if (lane == 0) a.near[row] = near ? 1 : 0;
    if (NTR > 64 && lane == 0) bcast[sub][2] = near ? 1.f : 0.f;
  }
  sync();
  if (NTR > 64) Q = bcast[sub][0], H = bcast[sub][1], near = a.near != nullptr && bcast[sub][2] != 0.f;
  if (near) return;  // all threads of the row: its results are distill_hot_kernel's
  const float g = a.g != nullptr ? a.g[row] : 1.f;
  float at, a1;
  dense_coeffs(a, g, Q, H, r, at, a1);
  if (tid < 64) {
    if (a.loss != nullptr) {
      const float loss = row_loss(a, lane, L, S, Q, H, r);
      if (lane == 0) a.loss[row] = loss;
    }
    if (lane == 0) {
      if (a.stats_out != nullptr) a.stats_out[row] = r;
      if (a.pred != nullptr) a.pred[row] = r.arg;
    }
    if (a.dz != nullptr) listed_grads(a, lane, L, twice, g, at, a1, m, S, H, r.st == 0.f, 0, K);
  }
  again();
  TO* dz = static_cast<TO*>(a.dz) + row * a.ldd;
  if (a.dz != nullptr) {
    typedef TO out_t __attribute__((ext_vector_type(V), aligned(sizeof(TO))));
    const int whole = K / (NTR * V);
    const float all = a.two ? at : at + a1;  // at T = 1 both softmaxes are one
    out_t last = {};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (v <= whole) {
        out_t o;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = raw[v][e] - m;
          float x = r.st == 0.f ? at : all * __builtin_amdgcn_exp2f(d * ct);
          if (a.two) x += a1 * __builtin_amdgcn_exp2f(d * c1);
          o[e] = (TO)x;
        }
        if (v < whole)
          *reinterpret_cast<out_t*>(elem(dz, (v * NTR + tid) * V)) = o;
        else
          last = o;
      }
    }
    const int i = (whole * NTR + tid) * V;
    if (i + V <= K) {
      *reinterpret_cast<out_t*>(elem(dz, i)) = last;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (i + e < K) *elem(dz, i + e) = last[e];
    }
  }
  if (a.dz == nullptr) return;
  sync();
  for (int j = tid; j <= a.k; j += NTR)
    if (L.keep[j] != 0) dz[L.cls[j]] = (TO)L.z[j];
}

// ---- rows cut into parts ------------------------------------------------------------------------
constexpr int PART_THREADS = 256;
constexpr int MAX_PARTS = 64;

__device__ __forceinline__ void merge_stats(RowStats& x, const RowStats& y, float ct, float c1) {
  const float m = fmaxf(x.m, y.m), mf = finite_max(m);
  const float fx = x.m - mf, fy = y.m - mf;
  x.st = x.st * __builtin_amdgcn_exp2f(fx * ct) + y.st * __builtin_amdgcn_exp2f(fy * ct);
  x.s1 = x.s1 * __builtin_amdgcn_exp2f(fx * c1) + y.s1 * __builtin_amdgcn_exp2f(fy * c1);
  x.arg = y.m > x.m || (y.m == x.m && y.arg < x.arg) ? y.arg : x.arg;
  x.m = m;
}

// The statistics of classes [c0, c1) of a row, by a block of NT threads; every thread of wave 0 gets
// them. c0 is a multiple of NT vectors.
template <class T, int NT>
__device__ __forceinline__ RowStats stream_stats(const Args& a, const T* z, int c0, int c1, RowStats* part) {
  constexpr int V = Vec<T>::N, U = 4, STEP = NT * V;
  const float ct = 1.44269504088896340736f / a.T, ce = 1.44269504088896340736f;
  RowStats r{-__builtin_inff(), 0.f, 0.f, 0};
#pragma unroll 1
  for (int base = c0; base < c1; base += U * STEP) {
    Held<T> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = base + u * STEP + (int)threadIdx.x * V;
      if (base + (u + 1) * STEP <= c1)
        raw[u].load(z, i);
      else
        raw[u].load(z, i, c1);
    }
    float m = r.m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) m = fmaxf(m, raw[u][e]);
    if (m > r.m) {  // rare after the first vectors
      if (a.pred != nullptr) {
        r.arg = a.K;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (raw[u][e] == m) r.arg = min(r.arg, base + u * STEP + (int)threadIdx.x * V + e);
      }
      r.st *= __builtin_amdgcn_exp2f((r.m - m) * ct);
      r.s1 *= __builtin_amdgcn_exp2f((r.m - m) * ce);
      r.m = m;
    }
    const float mf = finite_max(m);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) r.st += __builtin_amdgcn_exp2f((raw[u][e] - mf) * ct);
    if (a.two)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) r.s1 += __builtin_amdgcn_exp2f((raw[u][e] - mf) * ce);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const RowStats other{__shfl_xor(r.m, o, 64), __shfl_xor(r.st, o, 64), __shfl_xor(r.s1, o, 64),
                         __shfl_xor(r.arg, o, 64)};
    merge_stats(r, other, ct, ce);
  }
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = r;
  __syncthreads();
  r = part[0];
#pragma unroll 1
  for (int w = 1; w < NT / 64; ++w) merge_stats(r, part[w], ct, ce);
  if (!a.two) r.s1 = a.hard != 0.f ? r.st : 0.f;
  return r;
}

template <class T>
__global__ __launch_bounds__(PART_THREADS) void distill_parts_kernel(Args a, int len, RowStats* out) {
  __shared__ RowStats part[PART_THREADS / 64];
  const int64_t row = blockIdx.y;
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  const int c0 = blockIdx.x * len;
  const RowStats r = stream_stats<T, PART_THREADS>(a, z, c0, min(a.K, c0 + len), part);
  if (threadIdx.x == 0) out[row * gridDim.x + blockIdx.x] = r;
}

// The dense gradient of classes [c0, c1), last vectors first: what was read last is still near.
template <class T, class TO, int NT>
__device__ __forceinline__ void stream_grad(const Args& a, const T* z, TO* dz, int c0, int c1, RowStats r, float at,
                                            float a1) {
  constexpr int V = Vec<T>::N, U = 2, STEP = NT * V;
  typedef TO out_t __attribute__((ext_vector_type(V), aligned(sizeof(TO))));
  const float ct = 1.44269504088896340736f / a.T, ce = 1.44269504088896340736f, m = finite_max(r.m);
  const bool none = r.st == 0.f;
  const float all = a.two ? at : at + a1;  // at T = 1 both softmaxes are one
  const int steps = (c1 - c0 + U * STEP - 1) / (U * STEP);
  for (int s = steps - 1; s >= 0; --s) {
    const int base = c0 + s * U * STEP;
    Held<T> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = base + u * STEP + (int)threadIdx.x * V;
      if (base + (u + 1) * STEP <= c1)
        raw[u].load(z, i);
      else
        raw[u].load(z, i, c1);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = base + u * STEP + (int)threadIdx.x * V;
      out_t o;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = raw[u][e] - m;
        float x = none ? at : all * __builtin_amdgcn_exp2f(d * ct);
        if (a.two) x += a1 * __builtin_amdgcn_exp2f(d * ce);
        o[e] = (TO)x;
      }
      if (base + (u + 1) * STEP <= c1 || i + V <= c1) {
        *reinterpret_cast<out_t*>(elem(dz, i)) = o;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (i + e < c1) *elem(dz, i + e) = o[e];
      }
    }
  }
}

// loss, statistics and gradient from a row's (partial) statistics: one block per chunk of `len`
template <class T, class TO>
__global__ __launch_bounds__(PART_THREADS) void distill_chunks_kernel(Args a, int len) {
  __shared__ float bcast[2];
  extern __shared__ __attribute__((aligned(16))) unsigned char dyn[];
  const int64_t row = blockIdx.y;
  if (a.near != nullptr && !a.find && a.near[row] != 0) return;  // its results are distill_hot_kernel's
  const int lane = threadIdx.x & 63, cap = Listed::capacity(a.k);
  const float ct = 1.44269504088896340736f / a.T, ce = 1.44269504088896340736f;
  Listed L(dyn, cap);
  RowStats r = lane < a.parts ? a.stats_in[row * a.parts + lane] : RowStats{-__builtin_inff(), 0.f, 0.f, a.K};
  if (a.parts > 1) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const RowStats other{__shfl_xor(r.m, o, 64), __shfl_xor(r.st, o, 64), __shfl_xor(r.s1, o, 64),
                           __shfl_xor(r.arg, o, 64)};
      merge_stats(r, other, ct, ce);
    }
  } else {
    r = RowStats{__shfl(r.m, 0, 64), __shfl(r.st, 0, 64), __shfl(r.s1, 0, 64), __shfl(r.arg, 0, 64)};
  }
  const float m = finite_max(r.m), g = a.g != nullptr ? a.g[row] : 1.f;
  float S = 0.f, Q = 0.f, H = 0.f, at, a1;
  const int c0 = blockIdx.x * len, c1 = min(a.K, c0 + len);
  if (threadIdx.x < 64) {
    const bool twice = read_listed<T>(a, row, lane, L, S, Q, H);
    if (lane == 0) bcast[0] = Q, bcast[1] = H;
    dense_coeffs(a, g, Q, H, r, at, a1);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
    if (a.near != nullptr && a.find) {  // one block to a row, no gradient
      const bool near = near_rows(a, lane, L, S, r);
      if (lane == 0) a.near[row] = near ? 1 : 0;
      if (near) return;
    }
    if (blockIdx.x == 0) {
      if (a.loss != nullptr) {
        const float loss = row_loss(a, lane, L, S, Q, H, r);
        if (lane == 0) a.loss[row] = loss;
      }
      if (lane == 0) {
        if (a.stats_out != nullptr) a.stats_out[row] = r;
        if (a.pred != nullptr) a.pred[row] = r.arg;
      }
    }
    if (a.dz != nullptr) listed_grads(a, lane, L, twice, g, at, a1, m, S, H, r.st == 0.f, c0, c1);
  }
  if (a.dz == nullptr) return;
  __syncthreads();
  Q = bcast[0], H = bcast[1];
  dense_coeffs(a, g, Q, H, r, at, a1);
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  TO* dz = static_cast<TO*>(a.dz) + row * a.ldd;
  stream_grad<T, TO, PART_THREADS>(a, z, dz, c0, c1, r, at, a1);
  __syncthreads();
  for (int j = threadIdx.x; j <= a.k; j += PART_THREADS)
    if (L.keep[j] != 0) dz[L.cls[j]] = (TO)L.z[j];
}

// ---- high temperatures --------------------------------------------------------------------------
// A list of every class leaves p and q only (z - t) / T apart, while the loss, T^2 times a difference of their
// logarithms, stays of the size of (z - t)^2: what an f32 sum is off, about 2^-22, counts T^2 times (6e-5 at T = 16),
// and T times in the gradient of a listed class. Above, rows whose list holds nearly all of p (near_rows) are left out by
// the launches before, and their sums, listed classes and loss evaluated in 64 bits, T^2 2^-50; the dense part, where
// nothing cancels, is not. One block to a row, which it reads three times, the last two from the caches where it is not
// too long; bound by 64-bit exponentials, one a logit (two with labels). 256 x 1000 f32, all 1000 listed: 36 us, 18 at
// T = 16; 65536 x 1000 f32 of 16 listed, no row near: 127 us, 111 at T = 16; 7 x 200001 f32 of 33: 21 us, 15.
constexpr float HOT_T = 16.f;

// The listed classes of one row, in LDS: n = k entries, and the label as one more.
struct HotListed {
  double* q;       // exp((t_j - max t) / T), 0: absent
  int* cls;        // class, -1: absent
  float *t, *z;    // its logits; z later the whole gradient of the class
  uint16_t* keep;  // whether this entry writes it
  uint32_t* seen;  // as Listed's
  __device__ HotListed(unsigned char* lds, int cap) {
    q = reinterpret_cast<double*>(lds);
    cls = reinterpret_cast<int*>(q + cap);
    t = reinterpret_cast<float*>(cls + cap);
    z = t + cap;
    keep = reinterpret_cast<uint16_t*>(z + cap);
    seen = reinterpret_cast<uint32_t*>(keep + cap);
  }
  static __host__ __device__ size_t bytes(int k, int K) {
    return (size_t)Listed::capacity(k) * 22 + Listed::bits(k, K) / 8;
  }
};

template <class T, class TO, int NT>
__global__ __launch_bounds__(NT) void distill_hot_kernel(Args a) {
  constexpr int V = Vec<T>::N, STEP = NT * V;
  __shared__ double scratch[NT / 64];
  extern __shared__ __attribute__((aligned(16))) unsigned char dyn[];
  const int64_t row = blockIdx.x;
  if (a.near[row] == 0) return;
  const int K = a.K, k = a.k, tid = threadIdx.x, cap = Listed::capacity(k);
  const double rT = 1.0 / (double)a.T;
  const T* z = static_cast<const T*>(a.Z) + row * a.ldz;
  const int32_t* idx = a.idx + row * a.ldi;
  HotListed L(dyn, cap);
  auto sync = [] {
    if constexpr (NT > 64) {
      __syncthreads();
    } else {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  };
  auto fmax2 = [](float x, float y) { return fmaxf(x, y); };
  auto sum = [&](double v) {  // over the block, to all its threads
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    if constexpr (NT > 64) {
      __syncthreads();
      if ((tid & 63) == 0) scratch[tid >> 6] = v;
      __syncthreads();
      v = scratch[0];
#pragma unroll 1
      for (int w = 1; w < NT / 64; ++w) v += scratch[w];
      __syncthreads();
    }
    return v;
  };
  auto pass = [&](auto f) {  // f(logit, class); -inf past the row's end
    for (int i = tid * V; i < K; i += STEP) {
      Held<T> raw;
      raw.load(z, i, K);
#pragma unroll
      for (int e = 0; e < V; ++e) f(raw[e], i + e);
    }
  };
  // the list; what is found of it: a class out of range, a class that may stand twice, the label's
  constexpr int BAD = 1, TWICE = 2, LABEL = 4;
  float mt = -__builtin_inff();
  int found = 0;
  int label = a.hard != 0.f ? a.y[row] : -1;
  if (label >= K) found |= BAD, label = -1;
  const int bits = Listed::bits(k, K);
  for (int i = tid; i < bits / 32; i += NT) L.seen[i] = 0;
  sync();
  for (int j = tid; j < k; j += NT) {
    int c = idx[j];
    const float t = teacher_logit(a, row, j);
    if (c < 0 || t == -__builtin_inff()) c = -1;
    if (c >= K) found |= BAD, c = -1;
    L.cls[j] = c, L.t[j] = t, L.z[j] = c < 0 ? 0.f : (float)z[c];
    if (c < 0) continue;
    mt = fmaxf(mt, t);
    const uint32_t b = 1u << (c & 31);
    if (atomicOr(&L.seen[(c & (bits - 1)) >> 5], b) & b) found |= TWICE;
    if (c == label) found |= LABEL;
  }
  if (tid == 0) {
    L.z[k] = label < 0 ? 0.f : (float)z[label];
    for (int j = k; j < cap; ++j) L.cls[j] = j == k && label >= 0 ? label : -1, L.q[j] = 0.0;
  }
  sync();
  mt = finite_max(block_reduce<NT>(mt, reinterpret_cast<float*>(scratch), fmax2));
  found = block_reduce<NT>(found, reinterpret_cast<int*>(scratch), [](int x, int y) { return x | y; });
  double S = 0.0;
  for (int j = tid; j < k; j += NT) {
    const double q = L.cls[j] < 0 ? 0.0 : exp(((double)L.t[j] - (double)mt) * rT);
    L.q[j] = q;
    S += q;
  }
  S = sum(S);
  const double Q = (found & BAD) != 0 ? (double)__builtin_nanf("") : S == 0.0 ? 0.0 : S / S, H = label < 0 ? 0.0 : (double)a.hard;
  // the row
  RowStats r{-__builtin_inff(), 0.f, 0.f, 0};
  pass([&](float x, int) { r.m = fmaxf(r.m, x); });
  r.m = block_reduce<NT>(r.m, reinterpret_cast<float*>(scratch), fmax2);
  const double m = finite_max(r.m);
  double st = 0.0, s1 = 0.0;
  int arg = K;
  pass([&](float x, int i) {
    const double d = (double)x - m;
    st += exp(d * rT);
    if (a.hard != 0.f) s1 += exp(d);
    if (x == r.m) arg = min(arg, i);
  });
  st = sum(st), s1 = sum(s1);
  arg = block_reduce<NT>(arg, reinterpret_cast<int*>(scratch), [](int x, int y) { return min(x, y); });
  r.st = (float)st, r.s1 = (float)s1, r.arg = arg == K ? 0 : arg;
  const bool none = st == 0.0;
  if (a.loss != nullptr) {
    double part = 0.0;
    if (a.soft != 0.f && S != 0.0 && !none) {
      const double ratio = log(st / S);
      for (int j = tid; j < k; j += NT) {
        if (L.cls[j] < 0) continue;
        const double term = ((double)L.t[j] - (double)mt) * rT - ((double)L.z[j] - m) * rT + ratio;
        part += L.z[j] == -__builtin_inff() ? (double)__builtin_inff() : L.q[j] / S * term;
      }
    }
    double loss = sum(part) * (double)a.soft * (double)a.T * (double)a.T;
    if (!none && H != 0.0) loss += H * (log(s1) - ((double)L.z[k] - m));
    loss = none ? (Q != Q ? Q : 0.0) : loss + (Q - Q) + (st - st);
    if (tid == 0) a.loss[row] = (float)loss;
  }
  if (tid == 0) {
    if (a.stats_out != nullptr) a.stats_out[row] = r;
    if (a.pred != nullptr) a.pred[row] = r.arg;
  }
  if (a.dz == nullptr) return;
  const float g = a.g != nullptr ? a.g[row] : 1.f;
  const double soft = (double)a.soft * (double)a.T;
  sync();
  for (int j = tid; j <= k; j += NT) {
    const int c = L.cls[j];
    // a class that stands once writes itself, and takes the label along
    bool mine = c >= 0 && !(j == k && (found & LABEL) != 0);
    double q = L.q[j], hit = c == label ? 1.0 : 0.0;
    if ((found & TWICE) != 0) q = hit = 0.0;
    for (int i = 0; mine && (found & TWICE) != 0 && i < cap; i += 4) {  // its first entry sums all of it, in their order
      const int4 o = *reinterpret_cast<const int4*>(L.cls + i);
      const int oc[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (oc[e] == c) {
          if (i + e < j) mine = false;
          if (i + e == k)
            hit = 1.0;
          else
            q += L.q[i + e];
        }
    }
    L.keep[j] = mine ? 1 : 0;
    if (mine) {
      const double d = (double)L.z[j] - m;
      double v = none ? Q - Q : soft * (exp(d * rT) / st * Q - (S == 0.0 ? 0.0 : q / S));
      if (!none && H != 0.0) v += H * (exp(d) / s1 - hit);
      L.z[j] = (float)((double)g * v);
    }
  }
  float at, a1;
  dense_coeffs(a, g, (float)Q, (float)H, r, at, a1);
  TO* dz = static_cast<TO*>(a.dz) + row * a.ldd;
  sync();  // the listed logits have been read
  stream_grad<T, TO, NT>(a, z, dz, 0, K, r, at, a1);
  sync();
  for (int j = tid; j <= k; j += NT)
    if (L.keep[j] != 0) dz[L.cls[j]] = (TO)L.z[j];
}

// ---- host ---------------------------------------------------------------------------------------
// Rows [r0, r0 + rows) of a call.
template <class T, class TO>
Args rows_from(const Args& a, int64_t r0, int64_t rows) {
  Args b = a;
  b.B = rows;
  b.Z = static_cast<const T*>(a.Z) + r0 * a.ldz;
  b.idx = a.idx + r0 * a.ldi;
  b.t = static_cast<const char*>(a.t) + r0 * a.ldt * (int64_t)dtype_size(a.t_dt);
  if (a.y) b.y = a.y + r0;
  if (a.g) b.g = a.g + r0;
  if (a.loss) b.loss = a.loss + r0;
  if (a.pred) b.pred = a.pred + r0;
  if (a.stats_in) b.stats_in = a.stats_in + r0;
  if (a.stats_out) b.stats_out = a.stats_out + r0;
  if (a.dz) b.dz = static_cast<TO*>(a.dz) + r0 * a.ldd;
  if (a.near) b.near = a.near + r0;
  return b;
}

// Few threads for short rows, of whose blocks a CU holds many.
template <class T, class TO>
void launch_hot(const Args& a, hipStream_t stream) {
  const size_t lds = HotListed::bytes(a.k, a.K);
  const dim3 grid((unsigned)a.B);
  if (a.K <= 2048)
    hipLaunchKernelGGL((distill_hot_kernel<T, TO, 64>), grid, dim3(64), lds, stream, a);
  else if (a.K <= 16384)
    hipLaunchKernelGGL((distill_hot_kernel<T, TO, 256>), grid, dim3(256), lds, stream, a);
  else
    hipLaunchKernelGGL((distill_hot_kernel<T, TO, 1024>), grid, dim3(1024), lds, stream, a);
  MLAPI_HIP_CHECK(hipGetLastError());
}

template <class T, class TO, int NTR, int NV>
void launch_rows(const Args& a, hipStream_t stream) {
  constexpr int NT = NTR < 256 ? 256 : NTR, RPB = NT / NTR;
  const size_t lds = RPB * Listed::bytes(a.k, a.K);
  hipLaunchKernelGGL((distill_rows_kernel<T, TO, NTR, NV>), dim3((unsigned)((a.B + RPB - 1) / RPB)), dim3(NT), lds,
                     stream, a);
  MLAPI_HIP_CHECK(hipGetLastError());
}

struct Plan {
  int parts = 0;  // 0: whole rows in registers
  int len = 0;    // logits per part
};

constexpr int ROW_VECS = 1024 * 16;  // vectors that 1024 threads hold

// A row stays in registers where it fits: one read. Rows of more than 8192 vectors leave one block
// of 16 waves on a CU; up to 32 of them are cut into parts for more CUs than that (16 rows of 50000 f32: 10.9
// against 12.7 us; 64 rows: 16.2 against 15.2). Longer rows than registers hold are cut always.
template <class T>
Plan make_plan(int64_t B, int K) {
  Plan p;
  constexpr int STEP = PART_THREADS * Vec<T>::N;
  const int vecs = (K + Vec<T>::N - 1) / Vec<T>::N;
  if (vecs <= ROW_VECS / 2 || (vecs <= ROW_VECS && B > 32)) return p;
  // about 1024 blocks, each of at least four steps
  const int steps = (K + STEP - 1) / STEP;
  p.parts = (int)std::max<int64_t>(1, std::min<int64_t>({MAX_PARTS, (steps + 3) / 4, (1024 + B - 1) / B}));
  p.len = (steps + p.parts - 1) / p.parts * STEP;
  p.parts = (K + p.len - 1) / p.len;
  return p;
}

// The fewest threads per row, then the fewest vectors per thread, that hold the row: many small blocks on a
// CU let one row's loads run under another's exponentials. 8 vectors per thread fit 64 registers (two blocks
// of 1024 threads on a CU); 2048 rows of 65536 bf16 took 120 us so, 154 us when a compiler's choice of 88
// registers left one.
template <class T, class TO>
void launch_resident(const Args& a, hipStream_t stream) {
  const int vecs = (a.K + Vec<T>::N - 1) / Vec<T>::N;
  if (vecs <= 64) return launch_rows<T, TO, 64, 1>(a, stream);
  if (vecs <= 64 * 2) return launch_rows<T, TO, 64, 2>(a, stream);
  if (vecs <= 64 * 4) return launch_rows<T, TO, 64, 4>(a, stream);
  if (vecs <= 64 * 8) return launch_rows<T, TO, 64, 8>(a, stream);
  if (vecs <= 256 * 4) return launch_rows<T, TO, 256, 4>(a, stream);
  if (vecs <= 256 * 8) return launch_rows<T, TO, 256, 8>(a, stream);
  if (vecs <= 512 * 8) return launch_rows<T, TO, 512, 8>(a, stream);
  if (vecs <= 1024 * 8) return launch_rows<T, TO, 1024, 8>(a, stream);
  launch_rows<T, TO, 1024, 16>(a, stream);
}

template <class T, class TO>
void run_rows(Args a, RowStats* ws, hipStream_t stream) {
  const Plan p = make_plan<T>(a.B, a.K);
  a.find = true;
  if (p.parts == 0) {
    launch_resident<T, TO>(a, stream);
    if (a.near != nullptr) launch_hot<T, TO>(a, stream);
    return;
  }
  const size_t lds = Listed::bytes(a.k, a.K);
  a.parts = 1;
  for (int64_t r0 = 0; r0 < a.B; r0 += 65535) {  // grid.y holds 16 bits
    const unsigned rows = (unsigned)std::min<int64_t>(65535, a.B - r0);
    Args b = rows_from<T, TO>(a, r0, rows);
    if (!a.stats_in) {
      hipLaunchKernelGGL((distill_parts_kernel<T>), dim3((unsigned)p.parts, rows), dim3(PART_THREADS), 0, stream, b,
                         p.len, ws + r0 * p.parts);
      b.stats_in = ws + r0 * p.parts;
      b.parts = p.parts;
    }
    // the loss gathers logits of the whole row, and so does the search for near rows: where the gradient overwrites
    // them, or leaves such rows out, they go first
    const bool first = b.near != nullptr || (b.dz == b.Z && b.loss != nullptr);
    if (first) {
      Args l = b;
      l.dz = nullptr;
      hipLaunchKernelGGL((distill_chunks_kernel<T, TO>), dim3(1, rows), dim3(PART_THREADS), lds, stream, l, p.len);
      b.loss = nullptr, b.find = false;
    }
    if (!first || b.dz != nullptr)
      hipLaunchKernelGGL((distill_chunks_kernel<T, TO>), dim3(b.dz == nullptr ? 1u : (unsigned)p.parts, rows),
                         dim3(PART_THREADS), lds, stream, b, p.len);
    if (b.near != nullptr) launch_hot<T, TO>(rows_from<T, TO>(a, r0, rows), stream);
  }
  MLAPI_HIP_CHECK(hipGetLastError());
}

template <class T, class TO>
void run_distill(const Args& a, RowStats* ws, hipStream_t stream) {
  const int64_t step = logit_slice_rows(a.B);
  for (int64_t r0 = 0; r0 < a.B; r0 += step) run_rows<T, TO>(rows_from<T, TO>(a, r0, std::min(step, a.B - r0)), ws, stream);
}

}  // namespace

namespace {
size_t near_bytes(int64_t B, float T) { return T > HOT_T ? ((size_t)B * sizeof(int32_t) + 15) / 16 * 16 : 0; }
}  // namespace

size_t distill_workspace(int dt, int64_t B, int K, float temperature, bool stats_given) {
  if (B <= 0 || K < 1) return 0;
  const Plan p = dt == DT_F32 ? make_plan<float>(B, K) : make_plan<__bf16>(B, K);
  return near_bytes(B, temperature) + (stats_given ? 0 : (size_t)p.parts * (size_t)B * sizeof(RowStats));
}

void launch_distill(const DistillCall& c, hipStream_t stream) {
  if (c.B <= 0) return;
  if (c.K < 1 || c.K > LOGIT_MAX_CLASSES || c.k < 1 || c.k > LOGIT_MAX_TOP)
    throw std::invalid_argument("distill: 1 <= K <= 2^20 classes, 1 <= k <= 1024 entries");
  if (c.B > 0x7fffffff) throw std::invalid_argument("distill: more than 2^31 rows");
  if (!(c.temperature >= 1e-6f && c.temperature <= 1e6f))
    throw std::invalid_argument("distill: temperature in [1e-6, 1e6]");
  if (!(c.alpha >= 0.f && c.alpha <= 1.f)) throw std::invalid_argument("distill: alpha in [0, 1]");
  if (c.ldz < c.K || (c.dz != nullptr && c.ldd < c.K)) throw std::invalid_argument("distill: row stride below K");
  if (c.alpha != 1.f && c.y == nullptr) throw std::invalid_argument("distill: alpha below 1 needs labels");
  if (c.ws_bytes < distill_workspace(c.dt, c.B, c.K, c.temperature, c.stats_in != nullptr))
    throw std::invalid_argument("distill: workspace too small");
  Args a{};
  a.Z = c.Z, a.idx = c.idx, a.t = c.t, a.y = c.y, a.g = c.g, a.loss = c.loss, a.dz = c.dz, a.pred = c.pred;
  a.stats_in = static_cast<const RowStats*>(c.stats_in);
  a.stats_out = static_cast<RowStats*>(c.stats_out);
  a.B = c.B, a.ldz = c.ldz, a.ldi = c.ldi, a.ldt = c.ldt, a.ldd = c.ldd;
  a.K = c.K, a.k = c.k, a.parts = 1, a.t_dt = c.t_dt;
  a.T = c.temperature, a.soft = c.alpha, a.hard = c.y != nullptr ? 1.f - c.alpha : 0.f;
  a.two = a.hard != 0.f && c.temperature != 1.f;
  const size_t near = near_bytes(c.B, c.temperature);
  a.near = near != 0 ? static_cast<int32_t*>(c.workspace) : nullptr;
  RowStats* ws = reinterpret_cast<RowStats*>(static_cast<char*>(c.workspace) + near);
  if (c.dt == DT_F32 && c.out_dt == DT_F32) return run_distill<float, float>(a, ws, stream);
  if (c.dt == DT_F32 && c.out_dt == DT_BF16) return run_distill<float, __bf16>(a, ws, stream);
  if (c.dt == DT_BF16 && c.out_dt == DT_BF16) return run_distill<__bf16, __bf16>(a, ws, stream);
  if (c.dt == DT_F16 && c.out_dt == DT_F16) return run_distill<_Float16, _Float16>(a, ws, stream);
  throw std::invalid_argument("distill: logits f32, bf16 or f16; the gradient in their type (bf16 also of f32)");
}

}  // namespace mlapi
