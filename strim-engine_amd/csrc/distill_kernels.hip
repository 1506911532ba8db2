// distill_kernels.hip — distillation from a teacher's top logits.
#include "kernels.hpp"
#include "score.hpp"

namespace strim {

namespace {

constexpr int SC_T = 256;  // threads of a row's workgroup

template <int DT>
__device__ __forceinline__ float row_at(const void* row, int64_t v) {
  return DT == STRIM_DTYPE_BF16 ? bf16_to_f32(((const uint16_t*)row)[v]) : ((const float*)row)[v];
}
template <int DT>
__device__ __forceinline__ const void* row_of(const void* x, int64_t r, int64_t stride) {
  return (const char*)x + r * stride * (DT == STRIM_DTYPE_BF16 ? 2 : 4);
}
template <int DT>
__device__ __forceinline__ void row_set(void* row, int64_t v, float f) {
  if (DT == STRIM_DTYPE_BF16) ((uint16_t*)row)[v] = __builtin_bit_cast(uint16_t, (__bf16)f);
  else ((float*)row)[v] = f;
}
__device__ __forceinline__ bool allowed_at(const uint32_t* mask, int64_t v) {
  return !mask || ((mask[v >> 5] >> (v & 31)) & 1u);
}

// Block reductions; every thread gets the result. `op` merges b into a, in a fixed order.
template <class T, class Op>
__device__ __forceinline__ T block_all(T v, T* scratch, Op op) {
  const int t = threadIdx.x;
  __syncthreads();
  scratch[t] = v;
  for (int d = SC_T / 2; d > 0; d >>= 1) {
    __syncthreads();
    if (t < d) scratch[t] = op(scratch[t], scratch[t + d]);
  }
  __syncthreads();
  return scratch[0];
}

// max, sum exp((x - max) / T), sum (x - max) exp((x - max) / T); a max of -inf carries no sums (but
// keeps a NaN)
struct Stat {
  float m, s, u;
};
__device__ __forceinline__ Stat stat_merge(Stat a, Stat b, float c) {
  const float top = fmaxf(a.m, b.m);
  if (top == -INFINITY) return Stat{top, a.s + b.s, 0.0f};
  // (a difference that is the lowest value's would make u infinite, and that times 0)
  const float da = a.m == -INFINITY ? 0.0f : fmaxf(a.m - top, -1e30f);
  const float db = b.m == -INFINITY ? 0.0f : fmaxf(b.m - top, -1e30f);
  const float fa = __builtin_amdgcn_exp2f(da * c), fb = __builtin_amdgcn_exp2f(db * c);
  return Stat{top, a.s * fa + b.s * fb, (a.u + da * a.s) * fa + (b.u + db * b.s) * fb};
}
__device__ __forceinline__ void stat_add(Stat& a, float x, float c) {
  a = stat_merge(a, Stat{x, x == -INFINITY ? 0.0f : 1.0f + 0.0f * x, 0.0f}, c);
}

// A distillation row's numbers: from the statistics of its tokens (`tail`: of those that are no
// alternative) and its alternatives.
struct DistillRow {
  double lse, log_rest, loss, mass, r;
  bool has, bad;
};

template <int DT>
__device__ DistillRow distill_row(const DistillArgs& a, int64_t r, const void* row, bool given) {
  const int32_t* ids = a.ids + r * a.M;
  const float* lps = a.logprobs + r * a.M;
  DistillRow o{0.0, 0.0, 0.0, 0.0, 0.0, false, false};
  double tmax = -INFINITY;
  for (int m = 0; m < a.M; ++m) {
    if (ids[m] >= a.V) o.bad = true;
    if (ids[m] >= 0 && !(lps[m] == -INFINITY)) {
      o.has = true;
      tmax = fmax(tmax, (double)lps[m]);
    }
  }
  if (o.bad || !o.has) {
    o.has = false;
    return o;
  }
  if (a.tail) tmax = 0.0;
  double sum = 0.0;
  for (int m = 0; m < a.M; ++m)
    if (ids[m] >= 0 && !(lps[m] == -INFINITY)) sum += exp((double)lps[m] - tmax);
  o.mass = a.tail ? sum : 1.0;
  o.r = a.tail ? fmax(0.0, 1.0 - sum) : 0.0;
  if (given) {
    o.lse = a.lse[r];
    o.log_rest = a.log_rest ? a.log_rest[r] : 0.0;
    return o;
  }
  // (plain sums: one thread's worth of work per workgroup, repeated by all)
  __shared__ Stat s_stat[SC_T];
  const float c = 1.44269504088896340736f / a.T;
  Stat st{-INFINITY, 0.0f, 0.0f};
  for (int v = threadIdx.x; v < a.V; v += SC_T) {
    bool in = false;
    if (a.tail)
      for (int m = 0; m < a.M; ++m) in |= ids[m] == v && !(lps[m] == -INFINITY);
    if (!in) stat_add(st, row_at<DT>(row, v), c);
  }
  st = block_all(st, s_stat, [&](Stat p, Stat q) { return stat_merge(p, q, c); });
  double top = st.m;
  if (a.tail)
    for (int m = 0; m < a.M; ++m)
      if (ids[m] >= 0 && !(lps[m] == -INFINITY)) top = fmax(top, (double)row_at<DT>(row, ids[m]));
  double rest = st.m == -INFINITY ? st.s : (double)st.s * exp(((double)st.m - top) / a.T), in = 0.0;
  if (a.tail)
    for (int m = 0; m < a.M; ++m) {
      if (ids[m] < 0 || lps[m] == -INFINITY) continue;
      bool first = true;
      for (int q = 0; q < m; ++q) first &= !(ids[q] == ids[m] && !(lps[q] == -INFINITY));
      if (first) in += exp(((double)row_at<DT>(row, ids[m]) - top) / a.T);
    }
  const double ls = log(rest + in);
  o.lse = top / a.T + ls;
  o.log_rest = a.tail ? log(rest) - ls : 0.0;
  for (int m = 0; m < a.M; ++m) {
    if (ids[m] < 0 || lps[m] == -INFINITY) continue;
    const double lp = (double)lps[m] - tmax - (a.tail ? 0.0 : log(sum)), p = exp(lp);
    if (p > 0.0 || p != p) o.loss += p * (lp - (((double)row_at<DT>(row, ids[m]) - top) / a.T - ls));
  }
  if (o.r > 0.0) o.loss += o.r * (log(o.r) - o.log_rest);
  return o;
}

template <int DT, bool LOSS, bool GRAD>
__global__ __launch_bounds__(SC_T) void k_distill(DistillArgs a) {
  const int64_t r = blockIdx.x;
  const void* row = row_of<DT>(a.logits, r, a.stride);
  const DistillRow o = distill_row<DT>(a, r, row, !LOSS);
  if (LOSS && threadIdx.x == 0) {
    const float loss = (float)o.loss;
    a.loss[r] = loss;
    if (a.out_lse) a.out_lse[r] = (float)o.lse;
    if (a.out_log_rest) a.out_log_rest[r] = (float)o.log_rest;
    if (a.status)
      a.status[r] = o.bad ? STRIM_EINVAL : fabsf(loss) < INFINITY ? STRIM_OK : STRIM_ENONFINITE;
  }
  if (!GRAD) return;
  void* out = (void*)row_of<DT>(a.d_logits, r, a.d_stride);
  const int32_t* ids = a.ids + r * a.M;
  const float* lps = a.logprobs + r * a.M;
  double tmax = -INFINITY, sum = 0.0;
  if (a.tail) tmax = 0.0;
  else
    for (int m = 0; m < a.M; ++m)
      if (ids[m] >= 0 && !(lps[m] == -INFINITY)) tmax = fmax(tmax, (double)lps[m]);
  for (int m = 0; m < a.M; ++m)
    if (ids[m] >= 0 && !(lps[m] == -INFINITY)) sum += exp((double)lps[m] - tmax);
  if (a.tail) sum = 1.0;
  const double w = o.has ? (double)a.weights[r] / a.T : 0.0;
  const double in = w * (o.mass + o.r);
  const double other = o.r > 0.0 && o.log_rest > -1e300 ? in - w * o.r * exp(-o.log_rest) : in;
  for (int v = threadIdx.x; v < a.V; v += SC_T) {
    double d = 0.0;
    if (o.has && w != 0.0) {
      double p = 0.0;
      bool hit = false;
      for (int m = 0; m < a.M; ++m)
        if (ids[m] == v && !(lps[m] == -INFINITY)) {
          hit = true;
          p += exp((double)lps[m] - tmax) / sum;
        }
      const double q = exp((double)row_at<DT>(row, v) / a.T - o.lse);
      d = (hit || !a.tail ? in : other) * q - w * p;
    }
    row_set<DT>(out, v, (float)d);
  }
}

// (a factor of 1, what the last step of a backward pass usually has, costs no pass over the data)
template <int DT>
__global__ __launch_bounds__(SC_T) void k_distill_scale(void* data, int64_t n, const float* factor) {
  const float f = *factor;
  if (f == 1.0f) return;
  for (int64_t i = (int64_t)blockIdx.x * SC_T + threadIdx.x; i < n; i += (int64_t)gridDim.x * SC_T)
    row_set<DT>(data, i, row_at<DT>(data, i) * f);
}

}  // namespace

int64_t distill_workspace(int, int, int, bool) { return 0; }

hipError_t launch_distill(const DistillArgs& a, bool bf16, bool loss, bool grad, void*, hipStream_t st) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)a.N), dim3(SC_T), 0, st, a); };
  constexpr int B = STRIM_DTYPE_BF16, F = STRIM_DTYPE_F32;
  if (loss && grad) bf16 ? go(k_distill<B, true, true>) : go(k_distill<F, true, true>);
  else if (loss) bf16 ? go(k_distill<B, true, false>) : go(k_distill<F, true, false>);
  else bf16 ? go(k_distill<B, false, true>) : go(k_distill<F, false, true>);
  return hipGetLastError();
}

hipError_t launch_distill_scale(void* data, bool bf16, int64_t n, const float* factor, hipStream_t st) {
  const int64_t blocks = (n + SC_T - 1) / SC_T;
  const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192));
  if (bf16) hipLaunchKernelGGL(k_distill_scale<STRIM_DTYPE_BF16>, grid, dim3(SC_T), 0, st, data, n, factor);
  else hipLaunchKernelGGL(k_distill_scale<STRIM_DTYPE_F32>, grid, dim3(SC_T), 0, st, data, n, factor);
  return hipGetLastError();
}

}  // namespace strim
