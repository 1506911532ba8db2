// norm_kernels.hip — rows normalised by their root mean square or by mean and variance, and their
// gradients.
//
//   y = (x - mu) rstd w + b,  rstd = 1 / sqrt(mean (x - mu)^2 + eps),  mu = mean x or 0
//   with xh = (x - mu) rstd, h = w dy:
//   dx = rstd (h - xh mean(h xh) [- mean h]),  dw = sum_n dy xh,  db = sum_n dy
//
// A row is held in the registers of L threads, NV vectors of eight elements each: 16 lanes, a wave or a
// workgroup of 256 or 1,024, the fewest that hold it. The variance is taken of x - mu, not from the squares'
// mean. The weights' gradients are sums over the rows: each thread adds those of its own columns over the
// rows that its workgroup takes one after the other (the next row is requested before this one's sums are
// met), a workgroup leaves one float32 row of them, and k_norm_join adds those in order. Bound by HBM where rows are
// many (N = 4,096, K = 5,120, bf16: forward 20.5 us, 4.1 TB/s, backward with the weights' 27; 131,072 rows of 128: 13.7
// and 22.9), else by the launches (one row 3.1 us).
#include <type_traits>

#include "kernels.hpp"
#include "rows.hpp"
#include "score.hpp"

namespace strim {

namespace {

// A lane's eight columns from k0 on, as RowVec<DT, G> has a row's: of a weight or bias of either type (`none`
// where there is no tensor, 0 past K), and of a float32 row of sums.
template <int DT, int G, bool EVEN>
__device__ __forceinline__ void param8(const void* p, bool bf16, int k0, int lane, int K, float none, float (&f)[8]) {
  typedef RowVec<DT, G> X;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = none;
  if (!p) return;
  if (bf16 == X::BF16) {
    X v;
    v.template load_to<true, false, EVEN>((const char*)p, k0, lane, K);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = v.at(j);
    return;
  }
  const int k = k0 + X::first(lane);
  if (k + X::step(7) < K) {
    if constexpr (X::BF16) {  // float32 weights beside bf16 rows
      const ru32x4_any* a = (const ru32x4_any*)((const float*)p + k);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(a[j >> 2][j & 3]);
    } else {  // bf16 weights beside float32 rows
      typedef uint32_t pair_any __attribute__((ext_vector_type(2), aligned(2)));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const pair_any q = *(const pair_any*)((const uint16_t*)p + k + X::step(4 * i));
#pragma unroll
        for (int j = 0; j < 4; ++j)
          f[4 * i + j] = __uint_as_float(j & 1 ? q[j >> 1] & 0xFFFF0000u : q[j >> 1] << 16);
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    f[j] = 0.0f;
    const int at = k + X::step(j);
    if (at < K) f[j] = bf16 ? bf16_to_f32(((const uint16_t*)p)[at]) : ((const float*)p)[at];
  }
}
template <int DT, int G, bool EVEN>
__device__ __forceinline__ void sums8(float* out, int k0, int lane, int K, const float (&f)[8]) {
  typedef RowVec<DT, G> X;
  if constexpr (!X::BF16) {
    X v;
    v.set(f);
    v.template store_to<EVEN>((char*)out, k0, lane, K);
  } else {
    const int k = k0 + 8 * lane;
    if (k + 8 <= K) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *(ru32x4_any*)(out + k + 4 * i) =
            ru32x4{__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]),
                   __float_as_uint(f[4 * i + 3])};
      return;
    }
    if (EVEN) return;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < K) out[k + j] = f[j];
  }
}

// The sum of v over the row's L threads, in each of them. `scratch` (L > 64: a wave's place each) is free
// again after the next call's barrier, so two take turns.
template <int L>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
  if constexpr (L == 16) {
    v += dpp_f<DPP_XOR1>(v);
    v += dpp_f<DPP_XOR2>(v);
    v += dpp_f<DPP_HALF_MIRROR>(v);
    v += dpp_f<DPP_MIRROR>(v);
    return v;
  } else {
    v = wave_sum_f(v);
    if constexpr (L > WAVE) {
      if ((threadIdx.x & (WAVE - 1)) == 0) scratch[threadIdx.x / WAVE] = v;
      __syncthreads();
      v = scratch[0];
#pragma unroll
      for (int i = 1; i < L / WAVE; ++i) v += scratch[i];
    }
    return v;
  }
}

template <int L>
struct NormShape {
  static constexpr int T = L < 256 ? 256 : L;  // threads of a workgroup
  static constexpr int ROWS = T / L;           // rows it has at once
  static constexpr int G = L < WAVE ? L : WAVE;  // lanes that share a vector's columns
};

// How many workgroups of k_norm take the rows, as many as the chip holds at once, each the next row's loads on
// their way while it finishes one (N = 4,096, bf16: K = 5,120 23.0 -> 20.5 us, 8,192 33.7 -> 30.4, with mean 47.2 ->
// 36.3, 16,384 61.9 -> 52.5; 131,072 rows of 128 14.9 -> 13.8). 0: a workgroup for every row or four, for the
// shapes where that was as fast or faster (K = 1,024 with mean, N = 20,000: 20.6 us, against 22.4; float32, K =
// 6,000, N = 3,000: 30.1 against 33.4; 131,072 float32 rows of 128 25.4 against 26.9).
constexpr int norm_resident(int dt, int L, int NV) {
  const bool bf16 = dt == STRIM_DTYPE_BF16;
  return L == 1024 ? 256 : NV == 4 ? 512 : NV == 3 && bf16 ? 768 : NV == 1 && L <= WAVE && bf16 ? 2048 : 0;
}

// The weights as the rows' lanes hold them where both are of one type (`same`), asked for beside the row and
// not after its sums (N = 4,096, K = 5,120: 25.1 -> 23.0 us).
template <class X, int L, int NV, bool EVEN>
__device__ __forceinline__ void held_params(X (&w)[NV], const void* p, bool same, int g0, int lane, int K) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (p && same) w[i].template load_to<true, false, EVEN>((const char*)p, 8 * L * i + g0, lane, K);
}

template <int DT, int L, int NV, bool CENTER, bool EVEN>
__global__ __launch_bounds__(NormShape<L>::T) void k_norm(const NormArgs a, bool wbf16) {
  constexpr int ROWS = NormShape<L>::ROWS, G = NormShape<L>::G;
  constexpr bool AHEAD = norm_resident(DT, L, NV) > 0;
  typedef RowVec<DT, G> X;
  __shared__ float s_sum[2][2][16];
  const int l = threadIdx.x % L, lane = l % G, g0 = 8 * (l - lane);  // (of the row, of its group; the group's)
  const float inv = 1.0f / (float)a.K;
  const bool same = wbf16 == X::BF16;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  int64_t n = (int64_t)blockIdx.x * ROWS + threadIdx.x / L;
  X next[NV], wv[NV];
  auto request = [&](int64_t n) {
    const char* row = (const char*)a.x + n * a.x_stride * X::SIZE;
#pragma unroll
    for (int i = 0; i < NV; ++i) next[i].template load_to<true, false, EVEN>(row, 8 * L * i + g0, lane, a.K);
  };
  if (AHEAD && n < a.N) request(n);
  if (AHEAD) held_params<X, L, NV, EVEN>(wv, a.weight, same, g0, lane, a.K);
  for (int turn = 0; n < a.N; n += step, turn ^= 1) {
    if (!AHEAD) {
      request(n);
      held_params<X, L, NV, EVEN>(wv, a.weight, same, g0, lane, a.K);  // (beside the row, not after its sums)
    }
    X x[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = next[i];
    if (AHEAD && n + step < a.N) request(n + step);
    float mu = 0.0f;
    if constexpr (CENTER) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s += x[i].at(j);
      mu = row_sum<L>(s, s_sum[turn][0]) * inv;
    }
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int left = a.K - 8 * L * i - g0 - X::first(lane);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = !CENTER ? x[i].at(j) : (EVEN ? X::step(j & ~3) : X::step(j)) < left ? x[i].at(j) - mu : 0.0f;
        q = fma_f(c, c, q);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i].renew();
    const float rstd = 1.0f / sqrtf(row_sum<L>(q, s_sum[turn][1]) * inv + a.eps);
    char* out = (char*)a.y + n * a.y_stride * X::SIZE;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k0 = 8 * L * i + g0;
      float f[8], w[8], b[8];
      if (same) {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = a.weight ? wv[i].at(j) : 1.0f;
      } else {
        param8<DT, G, EVEN>(a.weight, wbf16, k0, lane, a.K, 1.0f, w);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = (x[i].at(j) - mu) * rstd;
      if (a.bias) {
        param8<DT, G, EVEN>(a.bias, wbf16, k0, lane, a.K, 0.0f, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = fma_f(f[j], w[j], b[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= w[j];
      }
      X y;
      y.set(f);
      y.template store_to<EVEN>(out, k0, lane, a.K);
    }
    if (l == 0) {
      if (a.rstd) a.rstd[n] = rstd;
      if (CENTER) a.mean[n] = mu;
    }
  }
}

// Rows too wide for registers: read again (from the caches) for each step. A workgroup of 1,024 a row.
template <int DT, bool CENTER>
__global__ __launch_bounds__(1024) void k_norm_wide(const NormArgs a, bool wbf16) {
  constexpr int T = 1024;
  typedef RowVec<DT> X;
  __shared__ float s_sum[2][2][16];
  const int lane = threadIdx.x & (WAVE - 1), g0 = 8 * WAVE * wave_id();
  const float inv = 1.0f / (float)a.K;
  int turn = 0;
  for (int64_t n = blockIdx.x; n < a.N; n += gridDim.x, turn ^= 1) {
    const char* row = (const char*)a.x + n * a.x_stride * X::SIZE;
    float mu = 0.0f, q = 0.0f;
    if constexpr (CENTER) {
      float s = 0.0f;
#pragma unroll 2
      for (int k0 = g0; k0 < a.K; k0 += 8 * T) {
        X x;
        x.template load_to<true>(row, k0, lane, a.K);
#pragma unroll
        for (int j = 0; j < 8; ++j) s += x.at(j);
      }
      mu = row_sum<T>(s, s_sum[turn][0]) * inv;
    }
#pragma unroll 2
    for (int k0 = g0; k0 < a.K; k0 += 8 * T) {
      X x;
      x.template load_to<true>(row, k0, lane, a.K);
      const int left = a.K - k0 - X::first(lane);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = !CENTER ? x.at(j) : X::step(j) < left ? x.at(j) - mu : 0.0f;
        q = fma_f(c, c, q);
      }
    }
    const float rstd = 1.0f / sqrtf(row_sum<T>(q, s_sum[turn][1]) * inv + a.eps);
    char* out = (char*)a.y + n * a.y_stride * X::SIZE;
    for (int k0 = g0; k0 < a.K; k0 += 8 * T) {
      X x;
      x.template load_to<true>(row, k0, lane, a.K);
      float f[8], w[8], b[8];
      param8<DT, WAVE, false>(a.weight, wbf16, k0, lane, a.K, 1.0f, w);
      param8<DT, WAVE, false>(a.bias, wbf16, k0, lane, a.K, 0.0f, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = fma_f((x.at(j) - mu) * rstd, w[j], b[j]);
      x.set(f);
      x.store_to(out, k0, lane, a.K);
    }
    if (threadIdx.x == 0) {
      if (a.rstd) a.rstd[n] = rstd;
      if (CENTER) a.mean[n] = mu;
    }
  }
}
template <int DT, bool CENTER>
__global__ __launch_bounds__(1024) void k_norm_grad_wide(const NormGradArgs a, bool wbf16) {
  constexpr int T = 1024;
  typedef RowVec<DT> X;
  __shared__ float s_sum[2][2][16];
  const int lane = threadIdx.x & (WAVE - 1), g0 = 8 * WAVE * wave_id();
  const float inv = 1.0f / (float)a.K;
  int turn = 0;
  for (int64_t n = blockIdx.x; n < a.N; n += gridDim.x, turn ^= 1) {
    const char* xr = (const char*)a.x + n * a.x_stride * X::SIZE;
    const char* gr = (const char*)a.dy + n * a.dy_stride * X::SIZE;
    char* out = (char*)a.dx + n * a.dx_stride * X::SIZE;
    const float rstd = a.rstd[n], mu = CENTER ? a.mean[n] : 0.0f;
    // xh, h of eight columns
    auto each = [&](int k0, float (&xh)[8], float (&h)[8]) {
      X x, g;
      x.template load_to<true>(xr, k0, lane, a.K);
      g.template load_to<true>(gr, k0, lane, a.K);
      param8<DT, WAVE, false>(a.weight, wbf16, k0, lane, a.K, 1.0f, h);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xh[j] = (x.at(j) - mu) * rstd;
        h[j] *= g.at(j);
      }
    };
    float c1 = 0.0f, c2 = 0.0f;
    for (int k0 = g0; k0 < a.K; k0 += 8 * T) {
      float xh[8], h[8];
      each(k0, xh, h);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        c1 = fma_f(h[j], xh[j], c1);
        c2 += h[j];
      }
    }
    c1 = row_sum<T>(c1, s_sum[turn][0]) * inv;
    c2 = CENTER ? row_sum<T>(c2, s_sum[turn][1]) * inv : 0.0f;
    for (int k0 = g0; k0 < a.K; k0 += 8 * T) {
      float xh[8], h[8];
      each(k0, xh, h);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = rstd * (fma_f(-xh[j], c1, h[j]) - c2);
      X y;
      y.set(h);
      y.store_to(out, k0, lane, a.K);
    }
  }
}

// PARAM 1: also the workgroup's sums of dy xh, to row blockIdx.x of `part` [grid][PARAM][K]; 2: of dy too.
// (Past K dy is 0, so that nothing there counts.)
template <int DT, int L, int NV, bool CENTER, int PARAM, bool EVEN>
__global__ __launch_bounds__(NormShape<L>::T) void k_norm_grad(const NormGradArgs a, bool wbf16, float* part) {
  constexpr int ROWS = NormShape<L>::ROWS, G = NormShape<L>::G;
  typedef RowVec<DT, G> X;
  __shared__ float s_sum[2][2][16];
  const int l = threadIdx.x % L, lane = l % G, g0 = 8 * (l - lane);
  const float inv = 1.0f / (float)a.K;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  X nx[NV], ng[NV];
  float nr = 0.0f, nm = 0.0f;
  auto request = [&](int64_t n) {
    const char* x = (const char*)a.x + n * a.x_stride * X::SIZE;
    const char* g = (const char*)a.dy + n * a.dy_stride * X::SIZE;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      nx[i].template load_to<true, false, EVEN>(x, 8 * L * i + g0, lane, a.K);
      ng[i].template load_to<true, false, EVEN>(g, 8 * L * i + g0, lane, a.K);
    }
    nr = a.rstd[n];
    if (CENTER) nm = a.mean[n];
  };
  int64_t n = (int64_t)blockIdx.x * ROWS + threadIdx.x / L;
  if (PARAM && n < a.N) request(n);
  // (without the sums each workgroup has a row of its own: the weights are read where they are used)
  float held[PARAM ? NV : 1][8], dw[PARAM > 0 ? NV : 1][8], db[PARAM > 1 ? NV : 1][8];
  auto weight = [&](int i, float (&w)[8]) {
    if constexpr (PARAM > 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = held[i][j];
    } else {
      param8<DT, G, EVEN>(a.weight, wbf16, 8 * L * i + g0, lane, a.K, 1.0f, w);
    }
  };
  if constexpr (PARAM > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      param8<DT, G, EVEN>(a.weight, wbf16, 8 * L * i + g0, lane, a.K, 1.0f, held[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        dw[i][j] = 0.0f;
        if (PARAM > 1) db[i][j] = 0.0f;
      }
    }
  }
  for (int turn = 0; n < a.N; n += step, turn ^= 1) {
    if (!PARAM) request(n);
    X x[NV], g[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i] = nx[i];
      g[i] = ng[i];
    }
    const float rstd = nr, mu = nm;
    if (PARAM && n + step < a.N) request(n + step);
    float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
      weight(i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = g[i].at(j), xh = (x[i].at(j) - mu) * rstd, h = d * w[j];
        c1 = fma_f(h, xh, c1);
        if (CENTER) c2 += h;
        if constexpr (PARAM > 0) dw[i][j] = fma_f(d, xh, dw[i][j]);
        if constexpr (PARAM > 1) db[i][j] += d;
      }
    }
    if (!a.dx) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i].renew();
      g[i].renew();
    }
    // (both sums at one barrier)
    if constexpr (L > WAVE) {
      c1 = wave_sum_f(c1);
      if (CENTER) c2 = wave_sum_f(c2);
      float* s = s_sum[turn][0];
      if ((threadIdx.x & (WAVE - 1)) == 0) {
        s[threadIdx.x / WAVE] = c1;
        s[16 + threadIdx.x / WAVE] = c2;
      }
      __syncthreads();
      c1 = s[0];
      c2 = s[16];
#pragma unroll
      for (int i = 1; i < L / WAVE; ++i) {
        c1 += s[i];
        c2 += s[16 + i];
      }
    } else {
      c1 = row_sum<L>(c1, nullptr);
      if (CENTER) c2 = row_sum<L>(c2, nullptr);
    }
    c1 *= inv;
    c2 = CENTER ? c2 * inv : 0.0f;
    char* out = (char*)a.dx + n * a.dx_stride * X::SIZE;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8], d[8];
      weight(i, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float xh = (x[i].at(j) - mu) * rstd, h = g[i].at(j) * w[j];
        d[j] = rstd * (fma_f(-xh, c1, h) - c2);
      }
      X y;
      y.set(d);
      y.template store_to<EVEN>(out, 8 * L * i + g0, lane, a.K);
    }
  }
  if constexpr (PARAM > 0) {
    float* out = part + (int64_t)blockIdx.x * PARAM * a.K;
    if constexpr (ROWS > 1) {
      // the workgroup's rows first
      __shared__ float s_acc[ROWS][8 * L * NV];
#pragma unroll
      for (int h = 0; h < PARAM; ++h) {
        if (h) __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            s_acc[threadIdx.x / L][8 * L * i + g0 + X::first(lane) + X::step(j)] = h == 0 ? dw[i][j] : db[PARAM > 1 ? i : 0][j];
        __syncthreads();
        for (int k = threadIdx.x; k < a.K; k += NormShape<L>::T) {
          float s = 0.0f;
#pragma unroll
          for (int q = 0; q < ROWS; ++q) s += s_acc[q][k];
          out[h * a.K + k] = s;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        sums8<DT, G, EVEN>(out, 8 * L * i + g0, lane, a.K, dw[i]);
        if constexpr (PARAM > 1) sums8<DT, G, EVEN>(out + a.K, 8 * L * i + g0, lane, a.K, db[i]);
      }
    }
  }
}

// The weights' gradients alone, where a row is too wide to hold them beside it: eight columns a thread, the
// rows dealt to gridDim.y parts.
template <int DT, bool CENTER, int PARAM>
__global__ __launch_bounds__(256) void k_norm_columns(const NormGradArgs a, float* part) {
  const int lane = threadIdx.x & (WAVE - 1), k0 = 8 * WAVE * ((int)blockIdx.x * (256 / WAVE) + wave_id());
  if (k0 >= a.K) return;
  float dw[8] = {}, db[8] = {};
#pragma unroll 4
  for (int64_t n = blockIdx.y; n < a.N; n += gridDim.y) {
    RowVec<DT> x, g;
    x.template load_to<true>((const char*)a.x + n * a.x_stride * RowVec<DT>::SIZE, k0, lane, a.K);
    g.template load_to<true>((const char*)a.dy + n * a.dy_stride * RowVec<DT>::SIZE, k0, lane, a.K);
    const float rstd = a.rstd[n], mu = CENTER ? a.mean[n] : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      dw[j] = fma_f(g.at(j), (x.at(j) - mu) * rstd, dw[j]);
      if (PARAM > 1) db[j] += g.at(j);
    }
  }
  float* out = part + (int64_t)blockIdx.y * PARAM * a.K;
  sums8<DT, WAVE, false>(out, k0, lane, a.K, dw);
  if constexpr (PARAM > 1) sums8<DT, WAVE, false>(out + a.K, k0, lane, a.K, db);
}

// dw and db from the workgroups' rows of `width` sums (K of dw, then K of db), added in order: 64 columns a
// workgroup, its waves a part of the rows each.
constexpr int NJ_T = 1024;
__global__ __launch_bounds__(NJ_T) void k_norm_join(const float* part, int parts, int width, int K, void* dw,
                                                    void* db, bool wbf16) {
  __shared__ float s_sum[NJ_T / WAVE][WAVE];
  const int lane = threadIdx.x & (WAVE - 1), wave = wave_id();
  const int at = blockIdx.x * WAVE + lane;
  float s = 0.0f;
  if (at < width) {
    const int each = (parts + NJ_T / WAVE - 1) / (NJ_T / WAVE);
    const int end = min(parts, (wave + 1) * each);
#pragma unroll 8
    for (int p = wave * each; p < end; ++p) s += part[(int64_t)p * width + at];
  }
  s_sum[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || at >= width) return;
#pragma unroll
  for (int i = 1; i < NJ_T / WAVE; ++i) s += s_sum[i][lane];
  void* out = at < K ? dw : db;
  const int k = at < K ? at : at - K;
  if (!out) return;
  if (wbf16) ((uint16_t*)out)[k] = __builtin_bit_cast(uint16_t, (__bf16)s);
  else ((float*)out)[k] = s;
}

__global__ __launch_bounds__(256) void k_norm_zero(int K, void* dw, void* db, bool wbf16) {
  const int k = blockIdx.x * 256 + threadIdx.x;
  if (k >= K) return;
  for (void* p : {dw, db})
    if (p) {
      if (wbf16) ((uint16_t*)p)[k] = 0;
      else ((float*)p)[k] = 0.0f;
    }
}

int64_t ceil_of(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The threads that hold a row, and their vectors, f(L, NV). False past what registers hold. Forward and
// backward in us at N = 20,000 with 4 vectors or fewer a lane of a wave a row, and with a workgroup a row:
// K = 1,024 19.6, 29.8 and 25.5, 40.6 (N = 1,100: 3.3, 7.7 and 3.6, 8.7), K = 2,048 37.8, 53.8 and 32.0, 52.5.
template <class F>
bool with_shape(int K, F f) {
  using std::integral_constant;
#define STRIM_SHAPE(L, NV)                                             \
  if (K <= 8 * L * NV) {                                               \
    f(integral_constant<int, L>{}, integral_constant<int, NV>{});      \
    return true;                                                       \
  }
  STRIM_SHAPE(16, 1)
  STRIM_SHAPE(64, 1)
  STRIM_SHAPE(64, 2)
  STRIM_SHAPE(256, 1)
  STRIM_SHAPE(256, 2)
  STRIM_SHAPE(256, 3)
  STRIM_SHAPE(256, 4)
  STRIM_SHAPE(1024, 2)
#undef STRIM_SHAPE
  return false;
}
constexpr int NO_WIDE = 8 * 256 * 4;  // columns past which the weights' gradients have a pass of their own
int rows_at_once(int K) {
  int rows = 1;
  with_shape(K, [&](auto l, auto) { rows = NormShape<decltype(l)::value>::ROWS; });
  return rows;
}

// Workgroups of the gradient's pass with the weights' sums: two a CU, or fewer with four rows each.
int norm_parts(int N, int K) {
  const int64_t groups = ceil_of(N, rows_at_once(K));
  if (K > NO_WIDE) return (int)(groups < 64 ? groups : 64);
  int64_t g = ceil_of(groups, 4);
  if (g < 128) g = groups < 128 ? groups : 128;
  return (int)(g < 512 ? g : 512);
}

template <class F>
void with_dtype(bool bf16, F f) {
  if (bf16) f(std::integral_constant<int, STRIM_DTYPE_BF16>{});
  else f(std::integral_constant<int, STRIM_DTYPE_F32>{});
}

}  // namespace

hipError_t launch_norm(const NormArgs& a, bool bf16, bool wbf16, hipStream_t st) {
  with_dtype(bf16, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    auto go = [&](auto kernel, int64_t groups, int64_t most, int threads) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)(groups < most ? groups : most)), dim3(threads), 0, st, a, wbf16);
    };
    const bool held = with_shape(a.K, [&](auto l, auto nv) {
      constexpr int L = decltype(l)::value, NV = decltype(nv)::value, T = NormShape<L>::T;
      const int64_t groups = ceil_of(a.N, NormShape<L>::ROWS);
      constexpr int64_t MOST = norm_resident(DT, L, NV) > 0 ? norm_resident(DT, L, NV) : 1 << 20;
      if (a.K % RowVec<DT>::RUN == 0)
        a.mean ? go(k_norm<DT, L, NV, true, true>, groups, MOST, T) : go(k_norm<DT, L, NV, false, true>, groups, MOST, T);
      else
        a.mean ? go(k_norm<DT, L, NV, true, false>, groups, MOST, T) : go(k_norm<DT, L, NV, false, false>, groups, MOST, T);
    });
    if (!held) a.mean ? go(k_norm_wide<DT, true>, a.N, 512, 1024) : go(k_norm_wide<DT, false>, a.N, 512, 1024);
  });
  return hipGetLastError();
}

int64_t norm_workspace(int N, int K, bool want_w, bool want_b) {
  return (int64_t)norm_parts(N, K) * (want_b ? 2 : want_w ? 1 : 0) * K * 4;
}

hipError_t launch_norm_grad(const NormGradArgs& a, bool bf16, bool wbf16, void* workspace, hipStream_t st) {
  const int param = a.db ? 2 : a.dw ? 1 : 0;  // rows of sums
  if (a.N == 0) {
    if (param)
      hipLaunchKernelGGL(k_norm_zero, dim3((unsigned)ceil_of(a.K, 256)), dim3(256), 0, st, a.K, a.dw, a.db, wbf16);
    return hipGetLastError();
  }
  float* part = (float*)workspace;
  const int parts = norm_parts(a.N, a.K);
  const bool wide = a.K > NO_WIDE;
  with_dtype(bf16, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (param && wide) {  // (before dx: it may go where x or dy is)
      const dim3 g((unsigned)ceil_of(a.K, 2048), (unsigned)parts);
      auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, dim3(256), 0, st, a, part); };
      if (a.mean) param > 1 ? go(k_norm_columns<DT, true, 2>) : go(k_norm_columns<DT, true, 1>);
      else param > 1 ? go(k_norm_columns<DT, false, 2>) : go(k_norm_columns<DT, false, 1>);
    }
    if (wide && !a.dx) return;
    auto go = [&](auto kernel, int64_t groups, int threads, auto... more) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)(groups < 1 << 20 ? groups : 1 << 20)), dim3(threads), 0, st, a, wbf16,
                         more...);
    };
    const bool held = with_shape(a.K, [&](auto l, auto nv) {
      constexpr int L = decltype(l)::value, NV = decltype(nv)::value, T = NormShape<L>::T;
      auto as = [&](auto center, auto even) {
        constexpr bool C = decltype(center)::value, E = decltype(even)::value;
        if constexpr (L < 1024) {
          if (param == 2) return go(k_norm_grad<DT, L, NV, C, 2, E>, parts, T, part);
          if (param == 1) return go(k_norm_grad<DT, L, NV, C, 1, E>, parts, T, part);
        }
        go(k_norm_grad<DT, L, NV, C, 0, E>, ceil_of(a.N, NormShape<L>::ROWS), T, part);
      };
      const bool even = a.K % RowVec<DT>::RUN == 0;
      if (a.mean) even ? as(std::true_type{}, std::true_type{}) : as(std::true_type{}, std::false_type{});
      else even ? as(std::false_type{}, std::true_type{}) : as(std::false_type{}, std::false_type{});
    });
    if (!held) a.mean ? go(k_norm_grad_wide<DT, true>, a.N, 1024) : go(k_norm_grad_wide<DT, false>, a.N, 1024);
  });
  if (param)
    hipLaunchKernelGGL(k_norm_join, dim3((unsigned)ceil_of((int64_t)param * a.K, WAVE)), dim3(NJ_T), 0, st, part, parts,
                       param * a.K, a.K, a.dw, a.db, wbf16);
  return hipGetLastError();
}

}  // namespace strim
