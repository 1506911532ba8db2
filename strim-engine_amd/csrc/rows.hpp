// rows.hpp — rows of logits as the scores and the distillation read and write them: eight tokens a
// lane, any alignment; and their softmax statistics.
#pragma once

#include "common.hpp"

namespace strim {

typedef uint32_t ru32x4 __attribute__((ext_vector_type(4)));
// (gfx950 takes 16-byte accesses at any address: rows of odd strides need no path of their own)
typedef ru32x4 ru32x4_any __attribute__((aligned(2)));
typedef float rf32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 rbf16x2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.44269504088896340736f;
constexpr uint32_t NINF_BITS = 0xFF800000u;

__device__ __forceinline__ float hw_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float fma_f(float a, float b, float c) { return __builtin_fmaf(a, b, c); }

// Eight tokens of a row as they lie in memory.
template <int DT>
struct RowVec {
  static constexpr int WORDS = DT == STRIM_DTYPE_BF16 ? 4 : 8;
  static constexpr int SIZE = DT == STRIM_DTYPE_BF16 ? 2 : 4;
  uint32_t w[WORDS];

  __device__ __forceinline__ float at(int j) const {
    if constexpr (DT == STRIM_DTYPE_BF16)
      return __uint_as_float(j & 1 ? w[j >> 1] & 0xFFFF0000u : w[j >> 1] << 16);
    else
      return __uint_as_float(w[j]);
  }
  // tokens v .. v + 7, all inside the row
  __device__ __forceinline__ void load(const char* row, int v) {
    const char* p = row + (int64_t)v * SIZE;
#pragma unroll
    for (int i = 0; i < WORDS / 4; ++i) {
      const ru32x4 q = ((const ru32x4_any*)p)[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[4 * i + j] = q[j];
    }
  }
  // tokens from v on that lie before V; past them -inf, or 0
  template <bool ZERO = false>
  __device__ __forceinline__ void load_to(const char* row, int v, int V) {
    if (v + 8 <= V) return load(row, v);
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = ZERO ? 0u : DT == STRIM_DTYPE_BF16 ? 0xFF80FF80u : NINF_BITS;
    const char* p = row + (int64_t)v * SIZE;
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (v + j < V) {
        if constexpr (DT == STRIM_DTYPE_BF16) {
          const uint32_t h = ((const uint16_t*)p)[j];
          w[j >> 1] = j & 1 ? (w[j >> 1] & 0xFFFFu) | h << 16 : (w[j >> 1] & 0xFFFF0000u) | h;
        } else {
          w[j] = ((const uint32_t*)p)[j];
        }
      }
  }
  // What was made of the words before is made anew after this (else the compiler keeps the tokens as floats
  // from one pass over a row to the next, beside the words, until registers spill).
  __device__ __forceinline__ void renew() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) asm volatile("" : "+v"(w[i]));
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
    if constexpr (DT == STRIM_DTYPE_BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rf32x2{f[2 * i], f[2 * i + 1]}, rbf16x2));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(f[i]);
    }
  }
  __device__ __forceinline__ void store_to(char* row, int v, int V) const {
    char* p = row + (int64_t)v * SIZE;
    if (v + 8 <= V) {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i)
        ((ru32x4_any*)p)[i] = ru32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
      return;
    }
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (v + j < V) {
        if constexpr (DT == STRIM_DTYPE_BF16) ((uint16_t*)p)[j] = (uint16_t)(w[j >> 1] >> (j & 1 ? 16 : 0));
        else ((uint32_t*)p)[j] = w[j];
      }
  }
};

template <int DT>
__device__ __forceinline__ float token_at(const char* row, int v) {
  return DT == STRIM_DTYPE_BF16 ? bf16_to_f32(((const uint16_t*)row)[v]) : ((const float*)row)[v];
}

__device__ __forceinline__ float op_add_f(float a, float b) { return a + b; }
__device__ __forceinline__ float wave_sum_f(float v) {
  STRIM_WAVE_REDUCE(float, v, dpp_f, rl_f, op_add_f);
  return v;
}

// Over some of a row's tokens: m the largest x, s = sum 2^y, u = sum y 2^y, with y = x c - b and c = log2(e) /
// T throughout. While tokens are added b is m c as it is rounded, so that a token costs one fused multiply-add;
// the rounding is the same for all of them, and stat_exact takes it out again (then y = (x - m) c). Without a
// token above -inf m is -inf, s = u = 0; a NaN or +inf makes s NaN.
struct RowStat {
  float m, s, u;
};
__device__ __forceinline__ float stat_ref(float m) { return m == -INFINITY ? 0.0f : m; }
// (past this m c or its difference to x c may be infinite: there y = (x - m) c from the start)
__device__ __forceinline__ bool stat_far(float ref) { return !(fabsf(ref) <= 1e30f); }
// a's sums for the maximum `top` >= a.m. (y is bounded: the type's lowest value lies 3.4e38 below zero, and u
// times a vanishing factor would be an infinity times 0.)
__device__ __forceinline__ void stat_rebase(RowStat& a, float top, float c) {
  const float ref = stat_ref(top);
  const float d = stat_far(ref) ? (a.m - ref) * c : a.m * c - ref * c, f = hw_exp2(d);
  a.u = a.s == 0.0f ? 0.0f : fma_f(fmaxf(d, -1e30f), a.s, a.u) * f;
  a.s = a.s == 0.0f ? 0.0f : a.s * f;
  a.m = top;
}
__device__ __forceinline__ void stat_merge(RowStat& a, RowStat b, float c) {
  const float top = fmaxf(a.m, b.m);
  stat_rebase(a, top, c);
  stat_rebase(b, top, c);
  a.s += b.s;
  a.u += b.u;
}
// A lane's next E tokens; `mx` is their maximum.
template <int E, bool U>
__device__ __forceinline__ void stat_add(RowStat& a, const float (&x)[E], float mx, float c) {
  if (mx > a.m) stat_rebase(a, mx, c);
  const float ref = stat_ref(a.m);
  auto one = [&](float y) {
    const float e = hw_exp2(y);  // (a NaN goes through to s)
    a.s += e;
    if (U) a.u = fma_f(fmaxf(y, -1e30f), e, a.u);
  };
  if (!stat_far(ref)) {
    const float b = -(ref * c);
#pragma unroll
    for (int j = 0; j < E; ++j) one(fma_f(x[j], c, b));
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) one((x[j] - ref) * c);
  }
}
// The wave's statistics in every lane.
__device__ __forceinline__ void stat_wave(RowStat& a, float c) {
  stat_rebase(a, wave_max_f(a.m), c);
  a.s = wave_sum_f(a.s);
  a.u = wave_sum_f(a.u);
}
// After the last merge.
__device__ __forceinline__ void stat_exact(RowStat& a, float c) {
  const float ref = stat_ref(a.m);
  if (stat_far(ref)) return;
  const float off = fma_f(ref, c, -(ref * c));  // m c past its rounding
  const float f = hw_exp2(-off);
  a.u = (a.u - off * a.s) * f;
  a.s *= f;
}

}  // namespace strim
