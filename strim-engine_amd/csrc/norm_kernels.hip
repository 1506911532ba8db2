// norm_kernels.hip — rows normalised by their root mean square or by mean and variance, and their
// gradients.
//
//   y = (x - mu) rstd w + b,  rstd = 1 / sqrt(mean (x - mu)^2 + eps),  mu = mean x or 0
//   with xh = (x - mu) rstd, h = w dy:
//   dx = rstd (h - xh mean(h xh) [- mean h]),  dw = sum_n dy xh,  db = sum_n dy
#include "kernels.hpp"
#include "score.hpp"

namespace strim {

namespace {

constexpr int NO_T = 256;

__device__ __forceinline__ float norm_at(const void* p, int64_t i, bool bf16) {
  return bf16 ? bf16_to_f32(((const uint16_t*)p)[i]) : ((const float*)p)[i];
}
__device__ __forceinline__ void norm_set(void* p, int64_t i, float f, bool bf16) {
  if (bf16) ((uint16_t*)p)[i] = __builtin_bit_cast(uint16_t, (__bf16)f);
  else ((float*)p)[i] = f;
}
__device__ __forceinline__ float norm_sum(float v, float* scratch) {
  __syncthreads();
  scratch[threadIdx.x] = v;
  for (int d = NO_T / 2; d > 0; d >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < d) scratch[threadIdx.x] += scratch[threadIdx.x + d];
  }
  __syncthreads();
  return scratch[0];
}

__global__ __launch_bounds__(NO_T) void k_norm(NormArgs a, bool bf16, bool wbf16) {
  __shared__ float s_sum[NO_T];
  const int64_t n = blockIdx.x;
  float mu = 0.0f;
  if (a.mean) {
    float s = 0.0f;
    for (int k = threadIdx.x; k < a.K; k += NO_T) s += norm_at(a.x, n * a.x_stride + k, bf16);
    mu = norm_sum(s, s_sum) / (float)a.K;
  }
  float q = 0.0f;
  for (int k = threadIdx.x; k < a.K; k += NO_T) {
    const float c = norm_at(a.x, n * a.x_stride + k, bf16) - mu;
    q += c * c;
  }
  const float rstd = 1.0f / sqrtf(norm_sum(q, s_sum) / (float)a.K + a.eps);
  for (int k = threadIdx.x; k < a.K; k += NO_T) {
    float y = (norm_at(a.x, n * a.x_stride + k, bf16) - mu) * rstd;
    if (a.weight) y *= norm_at(a.weight, k, wbf16);
    if (a.bias) y += norm_at(a.bias, k, wbf16);
    norm_set(a.y, n * a.y_stride + k, y, bf16);
  }
  if (threadIdx.x == 0) {
    if (a.rstd) a.rstd[n] = rstd;
    if (a.mean) a.mean[n] = mu;
  }
}

__global__ __launch_bounds__(NO_T) void k_norm_dx(NormGradArgs a, bool bf16, bool wbf16) {
  __shared__ float s_sum[NO_T];
  const int64_t n = blockIdx.x;
  const float rstd = a.rstd[n], mu = a.mean ? a.mean[n] : 0.0f;
  float c1 = 0.0f, c2 = 0.0f;
  for (int k = threadIdx.x; k < a.K; k += NO_T) {
    const float h = norm_at(a.dy, n * a.dy_stride + k, bf16) * (a.weight ? norm_at(a.weight, k, wbf16) : 1.0f);
    c1 += h * ((norm_at(a.x, n * a.x_stride + k, bf16) - mu) * rstd);
    c2 += h;
  }
  c1 = norm_sum(c1, s_sum) / (float)a.K;
  c2 = a.mean ? norm_sum(c2, s_sum) / (float)a.K : 0.0f;
  for (int k = threadIdx.x; k < a.K; k += NO_T) {
    const float h = norm_at(a.dy, n * a.dy_stride + k, bf16) * (a.weight ? norm_at(a.weight, k, wbf16) : 1.0f);
    const float xh = (norm_at(a.x, n * a.x_stride + k, bf16) - mu) * rstd;
    norm_set(a.dx, n * a.dx_stride + k, rstd * (h - xh * c1 - c2), bf16);
  }
}

__global__ __launch_bounds__(NO_T) void k_norm_dw(NormGradArgs a, bool bf16, bool wbf16) {
  const int64_t k = (int64_t)blockIdx.x * NO_T + threadIdx.x;
  if (k >= a.K) return;
  float w = 0.0f, b = 0.0f;
  for (int64_t n = 0; n < a.N; ++n) {
    const float g = norm_at(a.dy, n * a.dy_stride + k, bf16);
    w += g * ((norm_at(a.x, n * a.x_stride + k, bf16) - (a.mean ? a.mean[n] : 0.0f)) * a.rstd[n]);
    b += g;
  }
  if (a.dw) norm_set(a.dw, k, w, wbf16);
  if (a.db) norm_set(a.db, k, b, wbf16);
}

}  // namespace

hipError_t launch_norm(const NormArgs& a, bool bf16, bool wbf16, hipStream_t st) {
  hipLaunchKernelGGL(k_norm, dim3((unsigned)a.N), dim3(NO_T), 0, st, a, bf16, wbf16);
  return hipGetLastError();
}

int64_t norm_workspace(int, int, bool, bool) { return 0; }

hipError_t launch_norm_grad(const NormGradArgs& a, bool bf16, bool wbf16, void*, hipStream_t st) {
  if (a.dw || a.db)
    hipLaunchKernelGGL(k_norm_dw, dim3((unsigned)((a.K + NO_T - 1) / NO_T)), dim3(NO_T), 0, st, a, bf16, wbf16);
  if (a.dx && a.N > 0)
    hipLaunchKernelGGL(k_norm_dx, dim3((unsigned)a.N), dim3(NO_T), 0, st, a, bf16, wbf16);
  return hipGetLastError();
}

}  // namespace strim
