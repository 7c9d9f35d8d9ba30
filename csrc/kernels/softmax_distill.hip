// Distillation step of the multiclass trainer: the student is the linear model itself.
//
//   1. Z = X W^T + b, f32 [B, K] (the row-group MFMA kernel, gemm_softmax.hip);
//   2. loss rows and G = d(sum of losses)/dZ in bf16 [B, Kp] (distill.hip; the first maximum of each row beside them);
//   3. {loss, correct} sums of 1024 rows per block, in a fixed order;
//   4. dW_aug slabs = G^T X_aug (softmax_grad_wide.hip) and their deterministic sum with the SGD update.
//
// G is rounded to bf16 once, as the matrix product takes it (2^-8 of each entry at most); Z, the losses and
// all sums stay in f32. Z is written and read once more than the hard-label step's fused kernels need:
// the teacher's list enters between the two products.
#include <hip/hip_runtime.h>

#include <stdexcept>

#include "kernels/logit_rows.h"
#include "mlapi/common.h"
#include "mlapi/kernels.h"

namespace mlapi {
namespace {

constexpr int STAT_ROWS = 1024;

__global__ __launch_bounds__(256) void distill_stats_kernel(const float* loss, const int32_t* pred, const int32_t* y,
                                                            int64_t B, float* slabs) {
  __shared__ float scratch[4];
  const int64_t r0 = (int64_t)blockIdx.x * STAT_ROWS;
  float sum = 0.f, correct = 0.f;
  for (int64_t r = r0 + threadIdx.x; r < B && r < r0 + STAT_ROWS; r += 256) {
    sum += loss[r];
    if (y != nullptr && pred[r] == y[r]) correct += 1.f;
  }
  auto add = [](float a, float b) { return a + b; };
  sum = lrow::block_reduce<256>(sum, scratch, add);
  correct = lrow::block_reduce<256>(correct, scratch, add);
  if (threadIdx.x == 0) {
    slabs[2 * blockIdx.x] = sum;
    slabs[2 * blockIdx.x + 1] = correct;
  }
}

struct Layout {
  GtxPlan gtx;
  int stat_blocks;
  size_t z, g, slabs, stats, loss, pred, rows, total;
};

Layout make_layout(int64_t B, int K, int F) {
  Layout L{};
  L.gtx = gtx_plan(B, K, F);
  L.stat_blocks = (int)((B + STAT_ROWS - 1) / STAT_ROWS);
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t at = o;
    o = (o + bytes + 255) & ~size_t(255);
    return at;
  };
  L.z = take((size_t)B * K * sizeof(float));
  L.g = take((size_t)B * L.gtx.Kp * sizeof(uint16_t));
  L.slabs = take((size_t)L.gtx.row_groups * K * (F + 8) * sizeof(float));
  L.stats = take((size_t)L.stat_blocks * 2 * sizeof(float));
  L.loss = take((size_t)B * sizeof(float));
  L.pred = take((size_t)B * sizeof(int32_t));
  L.rows = take(distill_workspace(DT_F32, B, K, 1e6f));  // enough for every temperature
  L.total = o;
  return L;
}

}  // namespace

size_t softmax_distill_workspace(int64_t B, int K, int F) { return B <= 0 ? 0 : make_layout(B, K, F).total; }

void launch_softmax_distill(const void* X_aug, int64_t ldx, const void* W, const float* b, const int32_t* idx,
                            int64_t ldi, const void* t, int64_t ldt, int t_dt, int k, float temperature, float alpha,
                            const int32_t* y, int64_t B, int F, int K, float* dW_out, float* stats_out, void* workspace,
                            size_t ws_bytes, hipStream_t stream, const Sgd2D* update, P2PAllReduce* dp,
                            int dp_timeout_ms) {
  if (B <= 0) return;
  if (K < 2) throw std::invalid_argument("softmax_distill: at least 2 classes");
  if (ldx < F + 8 || ldx % 8 != 0)
    throw std::invalid_argument("softmax_distill: X_aug row stride must be >= F + 8 and a multiple of 8");
  if (update != nullptr && (update->params == nullptr || update->cols != F + 8 || update->pen_cols > F))
    throw std::invalid_argument("softmax_distill: fused update needs params [K, F + 8]");
  if (reinterpret_cast<uintptr_t>(X_aug) % 16 != 0 || reinterpret_cast<uintptr_t>(W) % 16 != 0)
    throw std::invalid_argument("softmax_distill: X_aug and W must be 16-byte aligned");
  const Layout L = make_layout(B, K, F);
  if (ws_bytes < L.total) throw std::invalid_argument("softmax_distill: workspace too small");
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  float* Z = reinterpret_cast<float*>(ws + L.z);
  uint16_t* G = reinterpret_cast<uint16_t*>(ws + L.g);
  launch_gemm_logits_ld(X_aug, ldx, W, b, B, F, K, Z, stream);
  DistillCall c;
  c.dt = DT_F32, c.out_dt = DT_BF16, c.t_dt = t_dt;
  c.Z = Z, c.ldz = K, c.idx = idx, c.ldi = ldi, c.t = t, c.ldt = ldt, c.k = k, c.y = y;
  c.loss = reinterpret_cast<float*>(ws + L.loss), c.pred = reinterpret_cast<int32_t*>(ws + L.pred);
  c.dz = G, c.ldd = L.gtx.Kp, c.B = B, c.K = K, c.temperature = temperature, c.alpha = alpha;
  c.workspace = ws + L.rows, c.ws_bytes = ws_bytes - L.rows;
  launch_distill(c, stream);
  float* stats = reinterpret_cast<float*>(ws + L.stats);
  hipLaunchKernelGGL(distill_stats_kernel, dim3((unsigned)L.stat_blocks), dim3(256), 0, stream, c.loss, c.pred, y, B,
                     stats);
  MLAPI_HIP_CHECK(hipGetLastError());
  float* slabs = reinterpret_cast<float*>(ws + L.slabs);
  launch_gtx(G, L.gtx, X_aug, ldx, B, F, K, slabs, stream);
  launch_gdw_reduce(slabs, L.gtx.row_groups, K, F + 8, dW_out, stats, L.stat_blocks, stats_out, update, dp,
                    dp_timeout_ms, stream);
}

}  // namespace mlapi
