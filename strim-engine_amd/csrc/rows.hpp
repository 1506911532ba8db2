// rows.hpp — rows of logits (and of hidden states) as the scores, the distillation and the norms read and
// write them: eight tokens a lane, any alignment; and their softmax statistics.
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

// Eight tokens a lane of the 8 G that G neighbouring lanes share, as they lie in memory: bf16, eight in a row;
// float32, two runs of four, 4 G tokens apart, so that the lanes' 16 bytes of one load are in a row as well
// (a lane's own 32 bytes by two loads: 4.6 TB/s past the caches, this 6.6).
template <int DT, int G = WAVE>
struct RowVec {
  static constexpr bool BF16 = DT == STRIM_DTYPE_BF16;
  static constexpr int WORDS = BF16 ? 4 : 8;
  static constexpr int SIZE = BF16 ? 2 : 4;
  static constexpr int RUN = BF16 ? 8 : 4;  // tokens in a row
  uint32_t w[WORDS];

  // where the lane's element j lies among the 8 G: first(lane) + step(j); and whose token `off` is
  static __device__ __forceinline__ int first(int lane) { return RUN * lane; }
  static constexpr __device__ __forceinline__ int step(int j) { return BF16 ? j : (j & 3) + (j >> 2) * 4 * G; }
  static __device__ __forceinline__ int lane_of(int off) { return BF16 ? off >> 3 : (off & (4 * G - 1)) >> 2; }
  static __device__ __forceinline__ int element_of(int off) { return BF16 ? off & 7 : (off & 3) + (off / (4 * G)) * 4; }

  __device__ __forceinline__ float at(int j) const {
    if constexpr (BF16)
      return __uint_as_float(j & 1 ? w[j >> 1] & 0xFFFF0000u : w[j >> 1] << 16);
    else
      return __uint_as_float(w[j]);
  }
  // The lane's of the tokens from v0 on, all inside the row. NT: past the caches.
  template <bool NT = false>
  __device__ __forceinline__ void load(const char* row, int v0, int lane) {
    const char* p = row + (int64_t)(v0 + first(lane)) * SIZE;
#pragma unroll
    for (int i = 0; i < WORDS / 4; ++i) {
      const ru32x4_any* a = (const ru32x4_any*)(p + i * 4 * G * SIZE);
      const ru32x4 q = NT ? __builtin_nontemporal_load(a) : *a;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[4 * i + j] = q[j];
    }
  }
  // Those that lie before V; past them -inf, or 0. EVEN: V is a multiple of RUN (less code, fewer registers).
  template <bool ZERO = false, bool NT = false, bool EVEN = false>
  __device__ __forceinline__ void load_to(const char* row, int v0, int lane, int V) {
    const int v = v0 + first(lane);
    const char* p = row + (int64_t)v * SIZE;
    if constexpr (EVEN) {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        constexpr uint32_t FILL = ZERO ? 0u : BF16 ? 0xFF80FF80u : NINF_BITS;
        ru32x4 q{FILL, FILL, FILL, FILL};
        const ru32x4_any* a = (const ru32x4_any*)(p + i * 4 * G * SIZE);
        if (v + step(4 * i) < V) q = NT ? __builtin_nontemporal_load(a) : *a;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[4 * i + j] = q[j];
      }
      return;
    }
    if (v + step(7) < V) return load<NT>(row, v0, lane);
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = ZERO ? 0u : BF16 ? 0xFF80FF80u : NINF_BITS;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (v + step(j) < V) {
        if constexpr (BF16) {
          const uint32_t h = ((const uint16_t*)p)[j];
          w[j >> 1] = j & 1 ? (w[j >> 1] & 0xFFFFu) | h << 16 : (w[j >> 1] & 0xFFFF0000u) | h;
        } else {
          w[j] = ((const uint32_t*)p)[step(j)];
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
    if constexpr (BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rf32x2{f[2 * i], f[2 * i + 1]}, rbf16x2));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(f[i]);
    }
  }
  template <bool EVEN = false>
  __device__ __forceinline__ void store_to(char* row, int v0, int lane, int V, bool nt = false) const {
    const int v = v0 + first(lane);
    char* p = row + (int64_t)v * SIZE;
    if (EVEN || v + step(7) < V) {
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i) {
        if (EVEN && v + step(4 * i) >= V) continue;
        const ru32x4 q{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
        ru32x4_any* a = (ru32x4_any*)(p + i * 4 * G * SIZE);
        if (nt) __builtin_nontemporal_store(q, a);
        else *a = q;
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (v + step(j) < V) {
        if constexpr (BF16) ((uint16_t*)p)[j] = (uint16_t)(w[j >> 1] >> (j & 1 ? 16 : 0));
        else ((uint32_t*)p)[step(j)] = w[j];
      }
  }
};

// The allow-mask's bits of a lane's eight tokens from v0 on (0 past V).
template <int DT>
__device__ __forceinline__ uint32_t allowed8(const uint32_t* mask, int v0, int lane, int V) {
  const uint8_t* b = (const uint8_t*)mask;
  const int v = v0 + RowVec<DT>::first(lane);
  if constexpr (DT == STRIM_DTYPE_BF16) {
    return v < V ? b[v >> 3] : 0u;
  } else {
    const int v2 = v + RowVec<DT>::step(4);
    const uint32_t lo = v < V ? b[v >> 3] >> (v & 4) : 0u, hi = v2 < V ? b[v2 >> 3] >> (v2 & 4) : 0u;
    return (lo & 15u) | (hi & 15u) << 4;
  }
}

// Stores of results larger than the memory-side cache go past the caches: nobody finds them there.
constexpr int64_t ROWS_CACHED = (int64_t)256 << 20;

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
// the rounding is the same for all of them, and stat_exact takes it out again (then y = (x - m) c). That holds
// while the rounding is small: it is half of m c's spacing, and from |m c| = 2^31 on it alone may pass 2^y's
// range. Past 2^20 (where it is 2^-5) y = (x - m) c from the start. Without a token above -inf m is -inf, s = u =
// 0; a NaN or +inf makes s NaN.
struct RowStat {
  float m, s, u;
};
__device__ __forceinline__ float stat_ref(float m) { return m == -INFINITY ? 0.0f : m; }
// (of m c: an infinite product or a NaN is far)
__device__ __forceinline__ bool stat_far(float mc) { return !(fabsf(mc) <= 0x1p20f); }
// a's sums for the maximum `top` >= a.m. (y is bounded: the type's lowest value lies 3.4e38 below zero, and u
// times a vanishing factor would be an infinity times 0.)
__device__ __forceinline__ void stat_rebase(RowStat& a, float top, float c) {
  const float ref = stat_ref(top), from = a.m * c, to = ref * c;
  float d = from - to;  // the old b less the new one, each as rounded or (far) exact
  if (stat_far(fmaxf(fabsf(from), fabsf(to)))) {
    if (!stat_far(to)) d = fma_f(a.m, c, -to);
    else d = stat_far(from) ? (a.m - ref) * c : fma_f(-ref, c, from);
  }
  const float f = hw_exp2(d);
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
  const float ref = stat_ref(a.m), mc = ref * c;
  auto one = [&](float y) {
    const float e = hw_exp2(y);  // (a NaN goes through to s)
    a.s += e;
    if (U) a.u = fma_f(fmaxf(y, -1e30f), e, a.u);
  };
  if (!stat_far(mc)) {
#pragma unroll
    for (int j = 0; j < E; ++j) one(fma_f(x[j], c, -mc));
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
  const float ref = stat_ref(a.m), mc = ref * c;
  if (stat_far(mc)) return;
  const float off = fma_f(ref, c, -mc);  // m c past its rounding
  const float f = hw_exp2(-off);
  a.u = (a.u - off * a.s) * f;
  a.s *= f;
}

}  // namespace strim
