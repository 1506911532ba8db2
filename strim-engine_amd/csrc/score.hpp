// score.hpp — arguments and launchers of the token scores, the distillation loss and the norms.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace strim {

struct ScoreArgs {
  const void* logits;
  int64_t stride;
  int32_t R, V;
  float T;
  const uint32_t* mask;  // [R][mask_stride] or null
  int64_t mask_stride;
  const int32_t* tokens;  // [R][S]
  int32_t S, ignore_index, top;
  float *logprobs, *entropy, *lse;
  int32_t* top_ids;
  float* top_logprobs;
  int32_t* status;
};

struct ScoreGradArgs {
  const void* logits;
  int64_t stride;
  int32_t R, V;
  float T;
  const uint32_t* mask;
  int64_t mask_stride;
  const int32_t* tokens;
  int32_t S, ignore_index;
  const float *lse, *entropy, *grad_logprobs, *grad_entropy, *grad_lse;
  void* d_logits;
  int64_t d_stride;
  bool stream;  // the launcher's: stores past the caches
};

struct DistillArgs {
  const void* logits;
  int64_t stride;
  int32_t N, V;
  float T;
  const int32_t* ids;     // [N][M]
  const float* logprobs;  // [N][M]
  int32_t M, tail;
  // the gradient alone: the forward call's; the loss: where they go (or null)
  const float *lse, *log_rest;
  float *out_lse, *out_log_rest, *loss;
  int32_t* status;
  const float* weights;  // the loss's gradient per row
  void* d_logits;
  int64_t d_stride;
  bool stream;  // the launcher's: stores past the caches
};

struct NormArgs {
  const void* x;
  int64_t x_stride;
  int32_t N, K;
  const void *weight, *bias;  // [K] or null
  float eps;
  void* y;
  int64_t y_stride;
  float *rstd, *mean;  // [N]; mean null: root mean square
};

struct NormGradArgs {
  const void* x;
  int64_t x_stride;
  const void* dy;
  int64_t dy_stride;
  int32_t N, K;
  const void* weight;
  const float *rstd, *mean;  // mean null: root mean square
  void* dx;                  // or null
  int64_t dx_stride;
  void *dw, *db;  // [K] or null
};

int64_t scores_workspace(int R, int V, int top);
hipError_t launch_scores(const ScoreArgs& a, bool bf16, void* workspace, hipStream_t st);
hipError_t launch_scores_grad(const ScoreGradArgs& a, bool bf16, hipStream_t st);
int64_t distill_workspace(int N, int V, int M, bool step);
hipError_t launch_distill(const DistillArgs& a, bool bf16, bool loss, bool grad, void* workspace,
                          hipStream_t st);
hipError_t launch_distill_scale(void* data, bool bf16, int64_t n, const float* factor, hipStream_t st);
hipError_t launch_norm(const NormArgs& a, bool bf16, bool wbf16, hipStream_t st);
int64_t norm_workspace(int N, int K, bool want_w, bool want_b);
hipError_t launch_norm_grad(const NormGradArgs& a, bool bf16, bool wbf16, void* workspace,
                            hipStream_t st);

}  // namespace strim
