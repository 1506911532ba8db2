// q4_kernels.hip — a vocabulary projection held in 4 bits with group scales: packing, reading
// back, and the logits of a few rows.
//
// Row v of [V, K] is K / 8 words of eight 4-bit codes, the lowest bits first, and per group of
// G consecutive elements (32, 64 or 128) a bf16 scale s and, unless the weights are symmetric,
// a bf16 bias b: the element is s q + b (symmetric: s (q - 8)).
//
//   logits[r][v] = sum over groups g of  s[v][g] T + (b[v][g] - 16 s[v][g]) X
//   T = sum over k in g of (16 + q[v][k]) x[r][k],   X = sum over k in g of x[r][k]
//
// 16 + q is made in place: a code moved to bits 3 .. 6 of a half word under the bits of 16.0
// in bf16, two codes an instruction pair (the shift, and an AND-OR), exact; no conversion, no
// scaling of weights before the product, so T is a bf16 MFMA's sum in float32, and a group
// costs two multiply-adds a result (one in k_q4_chunk, whose X term is MFMAs as well). The offset
// 16 (and not 128, which would save one of the four shifts) keeps what cancels between T and 16 X
// to a few bits. An infinity in a hidden row makes both infinite: its logits are NaN as a rule.
#include <atomic>

#include "kernels.hpp"

namespace strim {

typedef __bf16 qbf16x8 __attribute__((ext_vector_type(8)));
typedef float qf32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t qu32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t q4_bf16(float f) {
  const uint32_t u = __float_as_uint(f);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (u >> 16) | 0x0040u;
  return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}

// ---- packing ------------------------------------------------------------------------------
// Eight elements a thread, G / 8 neighbouring lanes a group; bound by HBM (V = 32,768, K = 5,120,
// groups of 64: bf16 95 us, 4.5 TB/s, float32 153, 5.0 TB/s). The words do not go past the caches:
// what reads them next finds them there (packed and read back, 8,193 x 2,048 in float32: 28 us, else
// 33).
//   biased:    s = bf16((max - min) r), b = bf16(min), q = clamp(rint((w - b) / s), 0, 15)
//   symmetric: s = bf16(max|w| r),                     q = clamp(rint(w / s) + 8, 0, 15)
// s and b are the values stored; s = 0 gives q = 0 (symmetric: 8). r is the float32 number next to
// 1 / 15 (1 / 7) and the product a float32 one, which is what torch's division of a float32 tensor
// by 15 (7) gives on the GPU: weights packed by elementary operations there have the same scales.
// The quotient itself may round to the other of two bf16 numbers that it is as good as between. A
// group with a NaN or an infinity gets NaN for its scale and its bias.
struct Q4Pack {
  const void* w;
  int64_t w_stride;
  int32_t V, K;
  uint32_t* words;
  uint16_t *scales, *biases;
};

// Largest (or least) of the lanes of a group of 4, 8 or 16, in every lane: neighbours, pairs,
// then the mirrored half rows and rows.
template <int LANES, bool MAX>
__device__ __forceinline__ float q4_extreme(float v) {
  auto with = [&](int other) {
    const float o = __int_as_float(other);
    v = MAX ? fmaxf(v, o) : fminf(v, o);
  };
  with(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xF, 0xF, false));  // 1 0 3 2
  with(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xF, 0xF, false));  // 2 3 0 1
  if constexpr (LANES > 4) with(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xF, 0xF, false));
  if constexpr (LANES > 8) with(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x140, 0xF, 0xF, false));
  return v;
}

// The items (row, E elements) that a thread takes: every `stride` of the whole.
template <int E>
struct Q4Walk {
  int64_t v, dv;
  int c, dc, per_row;
  __device__ __forceinline__ Q4Walk(int K) : per_row(K / E) {
    const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, stride = (int64_t)gridDim.x * 256;
    v = first / per_row, c = (int)(first - v * per_row);
    dv = stride / per_row, dc = (int)(stride - dv * per_row);
  }
  __device__ __forceinline__ void next() {
    v += dv, c += dc;
    if (c >= per_row) c -= per_row, ++v;
  }
};

template <int G, bool F32, bool SYM>
__global__ __launch_bounds__(256) void k_q4_pack(const Q4Pack a) {
  // (a group's lanes run together: K / 8 and the stride are multiples of G / 8, which divides a row
  // of 16 lanes)
  for (Q4Walk<8> at(a.K); at.v < a.V; at.next()) {
    const int64_t v = at.v;
    const int c = at.c;
    float x[8];
    if constexpr (F32) {
      const float4* p = (const float4*)((const float*)a.w + v * a.w_stride + 8 * c);
      const float4 lo = p[0], hi = p[1];
      x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w;
      x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
    } else {
      const qu32x4 d = *(const qu32x4*)((const uint16_t*)a.w + v * a.w_stride + 8 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = __uint_as_float(d[e] << 16);
        x[2 * e + 1] = __uint_as_float(d[e] & 0xFFFF0000u);
      }
    }
    float hi = SYM ? fabsf(x[0]) : x[0], lo = x[0], bad = 0.0f * x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      hi = fmaxf(hi, SYM ? fabsf(x[e]) : x[e]);
      lo = fminf(lo, x[e]);
      bad += 0.0f * x[e];  // NaN where an element is not finite
    }
    // (as an infinity, which the maximum carries on)
    if (!(bad == 0.0f)) hi = INFINITY;
    hi = q4_extreme<G / 8, true>(hi);
    if constexpr (!SYM) lo = q4_extreme<G / 8, false>(lo);
    const float nan = hi < INFINITY ? 0.0f : __uint_as_float(0x7FC00000u);
    const uint32_t s16 = q4_bf16((SYM ? hi * (1.0f / 7.0f) : (hi - lo) * (1.0f / 15.0f)) + nan);
    const uint32_t b16 = SYM ? 0u : q4_bf16(lo + nan);
    const float s = __uint_as_float(s16 << 16), b = __uint_as_float(b16 << 16);
    // The correctly rounded quotient from the correctly rounded reciprocal, with one correction
    // (Markstein's theorem; scales near the ends of the range divide instead), and its rounding to
    // an integer by a sum whose unit is one.
    constexpr float ONE = 12582912.0f;  // 1.5 2^23
    constexpr float LO = SYM ? -8.0f : 0.0f, HI = SYM ? 7.0f : 15.0f;
    float q[8];
    const bool plain = s == 0.0f || (s > 0x1p-60f && s < 0x1p60f);
    if (__ballot(!plain) == 0) {
      const float r = s > 0.0f ? 1.0f / s : 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = SYM ? x[e] : x[e] - b, t = d * r;
        q[e] = __builtin_fmaf(__builtin_fmaf(-t, s, d), r, t);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = s > 0.0f ? (SYM ? x[e] : x[e] - b) / s : 0.0f;
    }
    uint32_t word = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float n = fminf(fmaxf(q[e], LO), HI) + (ONE + (SYM ? 8.0f : 0.0f));
      word |= (__float_as_uint(n) & 15u) << (4 * e);
    }
    a.words[v * at.per_row + c] = word;
    if (c % (G / 8) == 0) {
      const int64_t g = v * (a.K / G) + c / (G / 8);
      a.scales[g] = (uint16_t)s16;
      if constexpr (!SYM) a.biases[g] = (uint16_t)b16;
    }
  }
}

// ---- reading back -------------------------------------------------------------------------
struct Q4Weights {
  const uint32_t* words;
  int64_t words_stride;  // words a row
  const uint16_t *scales, *biases;
  int64_t scales_stride;
  int32_t V, K;
};

// Sixteen bytes a thread, so that a store's lines are whole (float32, eight elements a thread: 3.6
// TB/s, four: 4.1), and past the caches (V = 32,768, K = 5,120, groups of 64: bf16 90 -> 67 us, 6.4
// TB/s; float32 185 -> 146, with a quarter of the workgroups 123, 6.2 TB/s, bf16 67 -> 76).
template <int G, bool F32>
__global__ __launch_bounds__(256) void k_q4_unpack(const Q4Weights a, void* out, int64_t out_stride) {
  constexpr int E = F32 ? 4 : 8;
  for (Q4Walk<E> at(a.K); at.v < a.V; at.next()) {
    const int64_t v = at.v;
    const int c = at.c;
    const uint32_t word = a.words[v * a.words_stride + c / (8 / E)] >> (F32 ? 16 * (c & 1) : 0);
    const int64_t g = v * a.scales_stride + c / (G / E);
    const float s = __uint_as_float((uint32_t)a.scales[g] << 16);
    const float b = a.biases ? __uint_as_float((uint32_t)a.biases[g] << 16) : 0.0f;
    const float z = a.biases ? 0.0f : 8.0f;
    float x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = ((float)((word >> (4 * e)) & 15u) - z) * s + b;
    if constexpr (F32) {
      __builtin_nontemporal_store(qf32x4{x[0], x[1], x[2], x[3]},
                                  (qf32x4*)((float*)out + v * out_stride + 4 * c));
    } else {
      qu32x4 d;
#pragma unroll
      for (int e = 0; e < 4; ++e) d[e] = q4_bf16(x[2 * e]) | (q4_bf16(x[2 * e + 1]) << 16);
      __builtin_nontemporal_store(d, (qu32x4*)((uint16_t*)out + v * out_stride + 8 * c));
    }
  }
}

// ---- logits -------------------------------------------------------------------------------
// A step is 128 elements of K: a 16-row weight tile's 16 lanes of row r each load 16 bytes (4
// words) in each quarter of the wave. An MFMA sums over the four quarters, so its four words
// must be of one group: wide groups (128) are as loaded, narrower ones are exchanged between
// the quarters (v_permlane32_swap; 32 also v_permlane16_swap), one or half an instruction a
// word. q4_koff says which elements of the step quarter h of MFMA t then holds.
template <int G>
__device__ __forceinline__ constexpr int q4_koff(int t, int h) {
  return G == 128 ? 32 * h + 8 * t
         : G == 64 ? 32 * (2 * (t >> 1) + (h & 1)) + 8 * (2 * (t & 1) + (h >> 1))
                   : 32 * t + 8 * h;
}

__device__ __forceinline__ void q4_swap32(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}
__device__ __forceinline__ void q4_swap16(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0], b = r[1];
}

// the words of MFMAs 0 .. 3 from a lane's four
template <int G>
__device__ __forceinline__ void q4_order(const qu32x4& w, uint32_t* o) {
  if constexpr (G == 128) {
    o[0] = w[0], o[1] = w[1], o[2] = w[2], o[3] = w[3];
  } else if constexpr (G == 64) {
    o[0] = w[0], o[2] = w[1], o[1] = w[2], o[3] = w[3];
    q4_swap32(o[0], o[2]);
    q4_swap32(o[1], o[3]);
  } else {
    uint32_t a = w[0], b = w[2], c = w[1], d = w[3];
    q4_swap32(a, b);
    q4_swap32(c, d);
    q4_swap16(a, c);
    q4_swap16(b, d);
    o[0] = a, o[1] = c, o[2] = b, o[3] = d;
  }
}

// The masks of q4_codes, in registers that the compiler does not know the values of: an
// instruction takes one literal, so that with known ones it makes two of each AND-OR.
struct Q4Masks {
  uint32_t codes, sixteen;
  __device__ __forceinline__ Q4Masks() {
    asm volatile("s_mov_b32 %0, 0x00780078" : "=s"(codes));
    asm volatile("v_mov_b32 %0, 0x41804180" : "=v"(sixteen));
  }
};

// 16 + q of a word's codes, in the order 0 4 1 5 2 6 3 7
__device__ __forceinline__ qbf16x8 q4_codes(uint32_t w, const Q4Masks& k) {
  const qu32x4 r = {((w << 3) & k.codes) | k.sixteen, ((w >> 1) & k.codes) | k.sixteen,
                    ((w >> 5) & k.codes) | k.sixteen, ((w >> 9) & k.codes) | k.sixteen};
  return __builtin_bit_cast(qbf16x8, r);
}

// eight elements of a hidden row in that order
__device__ __forceinline__ qu32x4 q4_interleave(const qu32x4& d) {
  return qu32x4{__builtin_amdgcn_perm(d[2], d[0], 0x05040100u), __builtin_amdgcn_perm(d[2], d[0], 0x07060302u),
                __builtin_amdgcn_perm(d[3], d[1], 0x05040100u), __builtin_amdgcn_perm(d[3], d[1], 0x07060302u)};
}

struct Q4Args {
  Q4Weights w;
  const uint16_t* x;   // hidden [B][x_stride]
  int64_t x_stride;
  int32_t B;
  uint8_t* blocks;     // k_q4_blocks: the hidden rows' fragments and group sums, by steps
  void* out;
  int64_t out_stride;
  int32_t out_f32;
  float* part;         // k_q4_chunk split along K: sums [split][B][V]
};

// Row of the batch at place m of an MFMA's 16: rows 0 .. 3 at places 0, 4, 8, 12, so that
// the results of up to 4 rows are one register a lane, of up to 8 two.
__device__ __forceinline__ int q4_row(int m) { return (m >> 2) + 4 * (m & 3); }

__device__ __forceinline__ void q4_store(const Q4Args& a, int b, int v, float y) {
  if (a.out_f32) ((float*)a.out)[(int64_t)b * a.out_stride + v] = y;
  else ((uint16_t*)a.out)[(int64_t)b * a.out_stride + v] = (uint16_t)q4_bf16(y);
}

// Sums X of a 16-place tile's fragments over a group: the product with ones.
__device__ __forceinline__ qf32x4 q4_sum(qu32x4 x, qf32x4 acc) {
  const qu32x4 one = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(qbf16x8, x),
                                                 __builtin_bit_cast(qbf16x8, one), acc, 0, 0, 0);
}

// The hidden rows by chunks of 512: per chunk 16 NT fragments of 1 KB (MFMA t of step s, batch tile
// nt, at (4 s + t) NT + nt, 16 bytes a lane), then the group sums as fragments too, of q4_chunk_sums
// MFMAs by the words of scales and biases that k_q4_chunk's lanes load for a chunk: even quarters
// scales, odd ones biases, eight groups (four and the same four again with groups of 128; with
// groups of 32 the upper quarters the second eight). Y = -16 X by scales, X by biases (symmetric:
// -24 X and 0) is in three bf16 parts that add up to its 24 bits: every product is exact. A workgroup
// a chunk and batch tile, a wave a step.
template <int G>
constexpr int q4_chunk_sums() {
  return 128 / G == 4 ? 3 : 128 / G;
}

template <int G, int NT>
__global__ __launch_bounds__(4 * WAVE) void k_q4_blocks(const Q4Args a) {
  constexpr int GPS = 128 / G, MPG = 4 / GPS, NS = q4_chunk_sums<G>();
  __shared__ float s_sum[4 * GPS][16];
  const int lane = threadIdx.x & (WAVE - 1), step = wave_id(), h = lane >> 4, m = lane & 15;
  const int nt = blockIdx.y, b = 16 * nt + q4_row(m);
  uint8_t* blk = a.blocks + (int64_t)blockIdx.x * (16 + NS) * NT * 1024 + lane * 16;
#pragma unroll
  for (int g = 0; g < GPS; ++g) {
    qf32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < MPG; ++q) {
      const int t = g * MPG + q, k = (blockIdx.x * 4 + step) * 128 + q4_koff<G>(t, h);
      qu32x4 x = {0u, 0u, 0u, 0u};
      if (b < a.B && k < a.w.K) x = q4_interleave(*(const qu32x4*)(a.x + (int64_t)b * a.x_stride + k));
      *(qu32x4*)(blk + ((4 * step + t) * NT + nt) * 1024) = x;
      s = q4_sum(x, s);
    }
    if (m == 0) *(qf32x4*)&s_sum[step * GPS + g][4 * h] = s;
  }
  __syncthreads();
  if (step >= NS) return;
  const bool sym = a.w.biases == nullptr;
  const float by = h & 1 ? (sym ? 0.0f : 1.0f) : sym ? -24.0f : -16.0f;
  qu32x4 y;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int g = G == 32 ? 8 * (h >> 1) + e : G == 64 ? e : e & 3;
    // which part: 3 none
    const int part = G == 32 ? step : G == 64 ? (step == 0 ? h >> 1 : h < 2 ? 2 : 3)
                                              : e < 4 ? (h < 2 ? 0 : 2) : h < 2 ? 1 : 3;
    float f = by * s_sum[g][m];
    uint32_t bits = q4_bf16(f);
    for (int d = 0; d < 2; ++d)
      if (d < part) f -= __uint_as_float(bits << 16), bits = q4_bf16(f);
    if (part == 3) bits = 0u;
    y[e / 2] = e & 1 ? y[e / 2] | bits << 16 : bits;
  }
  *(qu32x4*)(blk + ((16 + step) * NT + nt) * 1024) = y;
}

// Few rows: every workgroup keeps the hidden rows' fragments and sums X in LDS, whole, and its
// waves read their weights without meeting. A unit is four steps of a row tile; the workgroup's
// row tiles are one run of units, cut evenly between the waves, so a wave has whole tiles and at
// most a piece at either end. The pieces are added through LDS at the end, in the order of the
// waves. RB: result registers a lane that hold rows (1 or 2 for up to 4 or 8 rows). D: units in
// flight. WHOLE: K a multiple of a unit's 512; otherwise K of 8 groups or more. This form, with the
// weights through registers, is for scales that k_q4_dma cannot take (one row at V = 151,936,
// K = 5,120, groups of 64: 105 us, k_q4_dma 90).
//
// What bounds it is the address unit: lanes of one 16-byte load that are neighbours are in
// different rows, so each lane's piece is looked up by itself, 16 bytes a cycle. A unit's scales
// and biases therefore come by one such load (even quarters the scales, odd ones the biases,
// exchanged between the quarters afterwards) and not by one a step: with those it took 178 us.
constexpr int QS_NW = 16;
constexpr size_t QS_LDS = 160 * 1024;

template <int G, int RB>
constexpr int q4_step_bytes() {
  return 4 * 4 * 4 * RB * 16 + (128 / G) * 4 * RB * 4;  // fragments, then the sums
}

typedef uint32_t qu32x2u __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t qu32x4u __attribute__((ext_vector_type(4), aligned(2)));

template <int G, int RB, int D, bool WHOLE>
__global__ __launch_bounds__(QS_NW* WAVE, 4) void k_q4_stream(const Q4Args a, int tiles) {
  constexpr int GPS = 128 / G, MPG = 4 / GPS, ROWS = 4 * RB;
  constexpr int SW = G == 128 ? 2 : 4;  // words of scales a lane loads
  extern __shared__ __attribute__((aligned(16))) uint8_t s_all[];
  const int lane = threadIdx.x & (WAVE - 1), wv = wave_id(), h = lane >> 4, r16 = lane & 15;
  const int units = (a.w.K + 511) / 512, groups = a.w.K / G, pieces = a.w.K / 32;
  uint8_t* s_x = s_all;                                        // [step][MFMA][quarter][row] 16 B
  float* s_xs = (float*)(s_all + units * 4 * (16 * ROWS * 16));  // [group][row]
  float* s_part = s_xs + units * 4 * GPS * ROWS;               // [wave][2][RB][64]
  // this workgroup's tiles, and this wave's units of their run
  const int t0 = (int)((int64_t)blockIdx.x * tiles / gridDim.x);
  const int run = ((int)((int64_t)(blockIdx.x + 1) * tiles / gridDim.x) - t0) * units;
  const int first = run * wv / QS_NW, last = run * (wv + 1) / QS_NW;

  struct Unit {
    qu32x4 w[4];
    uint32_t s[SW];
  } buf[D];
  const bool sym = a.w.biases == nullptr;
  const uint16_t* side = (h & 1) && !sym ? a.w.biases : a.w.scales;
  // groups of 32: the upper quarters take a unit's second eight
  const int sofs = G == 32 ? 8 * (h >> 1) : 0;
  int lt = t0 + first / units, lu = first % units, at = first;  // the next request
  const uint32_t* wp;
  const uint16_t* sp;
  auto row = [&]() {
    const int v = min(lt * 16 + r16, a.w.V - 1);
    wp = a.w.words + (int64_t)v * a.w.words_stride + 64 * lu + 4 * h;
    sp = side + (int64_t)v * a.w.scales_stride + lu * 4 * GPS + sofs;
  };
  auto load = [&](Unit& u) {  // past the run's end: the last unit again
#pragma unroll
    for (int p = 0; p < 4; ++p)
      u.w[p] = *(const qu32x4*)(wp + (WHOLE ? 16 * p : min(16 * p, 4 * (pieces - 1 - 16 * lu - h))));
    const uint16_t* from = sp;
    // not past the row: an earlier run of scales, moved into place
    const int back = WHOLE ? 0 : max(0, lu * 4 * GPS + sofs + 2 * SW - groups);
    if constexpr (!WHOLE) from -= back;
    if constexpr (SW == 2) {
      const qu32x2u v = *(const qu32x2u*)from;
      u.s[0] = v[0], u.s[1] = v[1];
    } else {
      const qu32x4u v = *(const qu32x4u*)from;
      u.s[0] = v[0], u.s[1] = v[1], u.s[2] = v[2], u.s[3] = v[3];
    }
    if (++at < last) {
      wp += 64, sp += 4 * GPS;
      if (++lu == units) lu = 0, ++lt, row();
    }
  };
  row();
  if (first < last) {
#pragma unroll
    for (int d = 0; d < D; ++d) load(buf[d]);
  }

  // the hidden rows: lane = (quarter, place) of a step's four MFMAs
  for (int st = wv; st < units * 4; st += QS_NW) {
    const int m = r16, b = (m >> 2) + 4 * (m & (RB - 1));  // (the other places repeat these)
    const uint16_t* xr = a.x + (int64_t)min(b, a.B - 1) * a.x_stride;
    qu32x4 x[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) x[t] = *(const qu32x4*)(xr + min(st * 128 + q4_koff<G>(t, h), a.w.K - 8));
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const bool in = b < a.B && st * 128 + q4_koff<G>(t, h) < a.w.K;
      x[t] = q4_interleave(x[t]);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[t][e] = in ? x[t][e] : 0u;
      if ((m & 3) < RB) *(qu32x4*)(s_x + ((st * 4 + t) * 4 + h) * ROWS * 16 + b * 16) = x[t];
    }
#pragma unroll
    for (int g = 0; g < GPS; ++g) {
      qf32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < MPG; ++q) s = q4_sum(x[g * MPG + q], s);
      if (r16 == 0)
#pragma unroll
        for (int r = 0; r < RB; ++r) s_xs[(st * GPS + g) * ROWS + h + 4 * r] = s[r];
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

  const Q4Masks masks;
  const uint32_t keepb = sym ? 0u : 0xFFFFFFFFu;  // symmetric: no biases, and 8 less
  const float zero = sym ? -24.0f : -16.0f;
  const uint32_t xat = (uint32_t)(h * ROWS + (r16 >> 2) + 4 * (r16 & (RB - 1))) * 16;
  float acc[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) acc[r] = 0.0f;
  int ct = t0 + first / units, cu = first % units, from = cu, piece = 0;
  // lane: weight row r16 of the tile, rows h + 4 r
  auto finish = [&](bool whole) {
    const int v = ct * 16 + r16;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      if (!whole) s_part[((wv * 2 + piece) * RB + r) * WAVE + lane] = acc[r];
      else if (v < a.w.V && h + 4 * r < a.B) q4_store(a, h + 4 * r, v, acc[r]);
      acc[r] = 0.0f;
    }
    piece = 1;
  };
  auto compute = [&](Unit& u) {
    if constexpr (!WHOLE) {  // the scales moved back for want of room move into place
      const int back = max(0, cu * 4 * GPS + sofs + 2 * SW - groups);
#pragma unroll
      for (int d = SW / 2; d > 0; d /= 2)  // by d words
#pragma unroll
        for (int e = 0; e < SW; ++e)
          u.s[e] = back & (2 * d) ? (e + d < SW ? u.s[e + d] : 0u) : u.s[e];
      const bool whole_words = back >= 2 * SW;
#pragma unroll
      for (int e = 0; e < SW; ++e) {
        const uint32_t half = (u.s[e] >> 16) | (e + 1 < SW ? u.s[e + 1] << 16 : 0u);
        u.s[e] = whole_words ? 0u : back & 1 ? half : u.s[e];
      }
    }
    uint32_t sw[2 * GPS], bw[2 * GPS];  // the unit's scales and biases, in every quarter
#pragma unroll
    for (int e = 0; e < SW; ++e) {
      uint32_t s0 = u.s[e], b0 = u.s[e];
      q4_swap16(s0, b0);
      if constexpr (G == 32) {
        uint32_t s1 = s0, b1 = b0;
        q4_swap32(s0, s1);
        q4_swap32(b0, b1);
        sw[4 + e] = s1, bw[4 + e] = b1;
      }
      sw[e] = s0, bw[e] = b0;
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      uint32_t w[4];
      q4_order<G>(u.w[p], w);
#pragma unroll
      for (int g = 0; g < GPS; ++g) {
        const int i = p * GPS + g;
        const float sc = __uint_as_float(i & 1 ? sw[i / 2] & 0xFFFF0000u : sw[i / 2] << 16);
        const float bi = __uint_as_float((i & 1 ? bw[i / 2] & 0xFFFF0000u : bw[i / 2] << 16) & keepb);
        const float off = __builtin_fmaf(zero, sc, bi);
        qf32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < MPG; ++q) {
          const int m = g * MPG + q;
          const qu32x4 x = *(const qu32x4*)(s_x + ((cu * 4 + p) * 4 + m) * (4 * ROWS * 16) + xat);
          t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(qbf16x8, x),
                                                      q4_codes(w[m], masks), t, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          const float xs = s_xs[((cu * 4 + p) * GPS + g) * ROWS + h + 4 * r];
          acc[r] = __builtin_fmaf(sc, t[r], __builtin_fmaf(off, xs, acc[r]));
        }
      }
    }
    if (++cu == units) {
      finish(from == 0);
      cu = from = 0;
      ++ct;
    }
  };
  for (int i = first; i < last; i += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (i + d >= last) goto done;
      compute(buf[d]);
      load(buf[d]);
    }
  }
done:
  if (cu != from) finish(false);
  __syncthreads();
  // tiles that more than one wave has units of
  for (int t = wv; t * units < run; t += QS_NW) {
    const int b0 = t * units, b1 = b0 + units;  // its part of the run
    int w0 = (int)((int64_t)b0 * QS_NW / run);
    while (run * (w0 + 1) / QS_NW <= b0) ++w0;
    if (run * (w0 + 1) / QS_NW >= b1 && run * w0 / QS_NW <= b0) continue;
    float y[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) y[r] = 0.0f;
    for (int w = w0; w < QS_NW && run * w / QS_NW < b1; ++w) {
      if (run * (w + 1) / QS_NW == run * w / QS_NW) continue;
      const int p = run * w / QS_NW / units == t ? 0 : 1;  // the wave's first tile, or its last
#pragma unroll
      for (int r = 0; r < RB; ++r) y[r] += s_part[((w * 2 + p) * RB + r) * WAVE + lane];
    }
    const int v = (t0 + t) * 16 + r16;
#pragma unroll
    for (int r = 0; r < RB; ++r)
      if (v < a.w.V && h + 4 * r < a.B) q4_store(a, h + 4 * r, v, y[r]);
  }
}

// 64 lanes' 16 bytes each, straight to LDS from `lds` (the same in every lane) in lane order.
// ONCE: the lines are not read again.
template <bool ONCE>
__device__ __forceinline__ void q4_load_lds(uint32_t lds, const void* p) {
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt"
                 ::"s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(p) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 ::"s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(p) : "memory");
}

// k_q4_stream with the weights straight to LDS, each wave's two units in a ring of its own (as many
// waves as the hidden rows leave room for, six or more): an instruction's lanes take four rows of 256
// bytes, sixteen neighbours to a row, so the address unit no longer bounds it but HBM does (one row
// at V = 151,936, K = 5,120, groups of 64, 438 MB: 90 us, 5.7 of them the launch's start and end, the
// rest at 5.2 TB/s). A row's pieces lie in its place xor its number, where the waves' reads meet all
// banks evenly. The weights are marked as not read again: the scales' lines, read a piece at a time
// by unit after unit, stay in L2 (99 us and 493 MB from HBM without). An even number of groups, scales
// and biases 4-byte aligned, K of 8 groups or more.
template <int G, int RB, bool WHOLE>
__global__ __launch_bounds__(QS_NW* WAVE, 4) void k_q4_dma(const Q4Args a, int tiles) {
  constexpr int GPS = 128 / G, MPG = 4 / GPS, ROWS = 4 * RB;
  constexpr int GPW = G == 32 ? 8 : 4 * GPS;  // groups a lane's scale load is wanted for
  constexpr int UNIT = 5 * 1024;
  extern __shared__ __attribute__((aligned(1024))) uint8_t s_all[];
  const int lane = threadIdx.x & (WAVE - 1), wv = wave_id(), h = lane >> 4, r16 = lane & 15;
  const int nw = blockDim.x / WAVE;
  const int units = (a.w.K + 511) / 512, groups = a.w.K / G, pieces = a.w.K / 32;
  uint8_t* s_w = s_all + wv * 2 * UNIT;                        // this wave's two units
  uint8_t* s_x = s_all + nw * 2 * UNIT;                        // [step][MFMA][quarter][row] 16 B
  float* s_xs = (float*)(s_x + units * 4 * (16 * ROWS * 16));  // [group][row]
  float* s_part = (float*)s_all;                               // at the end: [wave][2][RB][64]
  const uint32_t ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)s_w;
  // this workgroup's tiles, and this wave's units of their run
  const int t0 = (int)((int64_t)blockIdx.x * tiles / gridDim.x);
  const int run = ((int)((int64_t)(blockIdx.x + 1) * tiles / gridDim.x) - t0) * units;
  const int first = run * wv / nw, last = run * (wv + 1) / nw;

  const bool sym = a.w.biases == nullptr;
  const uint16_t* side = (h & 1) && !sym ? a.w.biases : a.w.scales;
  const int sofs = G == 32 ? 8 * (h >> 1) : 0;  // the upper quarters: a unit's second eight
  int lt = t0 + first / units, lu = first % units;  // the next request
  auto load = [&](int slot) {
    const int v0 = lt * 16, most = a.w.V - 1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // four rows, 256 bytes of each
      const int r = 4 * j + h, c = 16 * lu + (r16 ^ r);
      q4_load_lds<true>(ring + slot * UNIT + j * 1024,
                  a.w.words + (int64_t)min(v0 + r, most) * a.w.words_stride +
                      4 * (WHOLE ? c : min(c, pieces - 1)));
    }
    const int g0 = lu * 4 * GPS + sofs;
    q4_load_lds<false>(ring + slot * UNIT + 4096, side + (int64_t)min(v0 + r16, most) * a.w.scales_stride +
                                               min(g0, groups - 8));
    if (++lu == units) lu = 0, ++lt;
  };
  if (first < last) load(0);
  if (first + 1 < last) load(1);

  // the hidden rows: lane = (quarter, place) of a step's four MFMAs
  for (int st = wv; st < units * 4; st += nw) {
    const int m = r16, b = (m >> 2) + 4 * (m & (RB - 1));  // (the other places repeat these)
    const uint16_t* xr = a.x + (int64_t)min(b, a.B - 1) * a.x_stride;
    qu32x4 x[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) x[t] = *(const qu32x4*)(xr + min(st * 128 + q4_koff<G>(t, h), a.w.K - 8));
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const bool in = b < a.B && st * 128 + q4_koff<G>(t, h) < a.w.K;
      x[t] = q4_interleave(x[t]);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[t][e] = in ? x[t][e] : 0u;
      if ((m & 3) < RB) *(qu32x4*)(s_x + ((st * 4 + t) * 4 + h) * ROWS * 16 + b * 16) = x[t];
    }
#pragma unroll
    for (int g = 0; g < GPS; ++g) {
      qf32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < MPG; ++q) s = q4_sum(x[g * MPG + q], s);
      if (r16 == 0)
#pragma unroll
        for (int r = 0; r < RB; ++r) s_xs[(st * GPS + g) * ROWS + h + 4 * r] = s[r];
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

  const Q4Masks masks;
  const uint32_t keepb = sym ? 0u : 0xFFFFFFFFu;  // symmetric: no biases, and 8 less
  const float zero = sym ? -24.0f : -16.0f;
  const uint32_t xat = (uint32_t)(h * ROWS + (r16 >> 2) + 4 * (r16 & (RB - 1))) * 16;
  float acc[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) acc[r] = 0.0f;
  float part[2][RB];  // pieces of the wave's first and last tile
  int ct = t0 + first / units, cu = first % units, from = cu, piece = 0;
  // lane: weight row r16 of the tile, rows h + 4 r
  auto finish = [&](bool whole) {
    const int v = ct * 16 + r16;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      if (!whole) part[piece][r] = acc[r];
      else if (v < a.w.V && h + 4 * r < a.B) q4_store(a, h + 4 * r, v, acc[r]);
      acc[r] = 0.0f;
    }
    piece = 1;
  };
  for (int i = first, slot = 0; i < last; ++i, slot ^= 1) {
    if (i + 1 < last) asm volatile("s_waitcnt vmcnt(5)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const uint8_t* u = s_w + slot * UNIT;
    qu32x4 wd[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) wd[p] = *(const qu32x4*)(u + r16 * 256 + (((4 * p + h) ^ r16) << 4));
    constexpr int SW = GPW / 2;  // words of scales from one lane's load
    uint32_t sw[2 * GPS], bw[2 * GPS];
#pragma unroll
    for (int half = 0; half < 2 * GPS / SW; ++half) {
      const uint32_t* sp = (const uint32_t*)(u + 4096 + (half * 32 + r16) * 16);
      if constexpr (WHOLE && SW == 4) {
        const qu32x4 s4 = *(const qu32x4*)sp, b4 = *(const qu32x4*)(sp + 64);
#pragma unroll
        for (int e = 0; e < 4; ++e) sw[4 * half + e] = s4[e], bw[4 * half + e] = b4[e];
      } else {
        // a load that would pass the row's end began earlier
        const int g0 = cu * 4 * GPS + 8 * half, back = max(0, g0 + 8 - groups) / 2;
#pragma unroll
        for (int e = 0; e < SW; ++e) {
          const bool in = g0 + 2 * e < groups;  // (an even number of groups)
          const uint32_t sv = sp[min(back + e, 3)], bv = sp[64 + min(back + e, 3)];
          sw[SW * half + e] = in ? sv : 0u;
          bw[SW * half + e] = in ? bv : 0u;
        }
      }
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      uint32_t w[4];
      q4_order<G>(wd[p], w);
#pragma unroll
      for (int g = 0; g < GPS; ++g) {
        const int n = p * GPS + g;
        const float sc = __uint_as_float(n & 1 ? sw[n / 2] & 0xFFFF0000u : sw[n / 2] << 16);
        const float bi = __uint_as_float((n & 1 ? bw[n / 2] & 0xFFFF0000u : bw[n / 2] << 16) & keepb);
        const float off = __builtin_fmaf(zero, sc, bi);
        qf32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < MPG; ++q) {
          const int m = g * MPG + q;
          const qu32x4 x = *(const qu32x4*)(s_x + ((cu * 4 + p) * 4 + m) * (4 * ROWS * 16) + xat);
          t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(qbf16x8, x),
                                                      q4_codes(w[m], masks), t, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          const float xs = s_xs[((cu * 4 + p) * GPS + g) * ROWS + h + 4 * r];
          acc[r] = __builtin_fmaf(sc, t[r], __builtin_fmaf(off, xs, acc[r]));
        }
      }
    }
    // every read of the slot has returned before it is filled again
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (i + 2 < last) load(slot);
    if (++cu == units) {
      finish(from == 0);
      cu = from = 0;
      ++ct;
    }
  }
  if (cu != from) finish(false);
  __syncthreads();  // the ring is free in every wave: it takes the pieces
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int r = 0; r < RB; ++r) s_part[((wv * 2 + q) * RB + r) * WAVE + lane] = part[q][r];
  __syncthreads();
  // tiles that more than one wave has units of
  for (int t = wv; t * units < run; t += nw) {
    const int b0 = t * units, b1 = b0 + units;  // its part of the run
    int w0 = (int)((int64_t)b0 * nw / run);
    while (run * (w0 + 1) / nw <= b0) ++w0;
    if (run * (w0 + 1) / nw >= b1 && run * w0 / nw <= b0) continue;
    float y[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) y[r] = 0.0f;
    for (int w = w0; w < nw && run * w / nw < b1; ++w) {
      if (run * (w + 1) / nw == run * w / nw) continue;
      const int q = run * w / nw / units == t ? 0 : 1;  // the wave's first tile, or its last
#pragma unroll
      for (int r = 0; r < RB; ++r) y[r] += s_part[((w * 2 + q) * RB + r) * WAVE + lane];
    }
    const int v = (t0 + t) * 16 + r16;
#pragma unroll
    for (int r = 0; r < RB; ++r)
      if (v < a.w.V && h + 4 * r < a.B) q4_store(a, h + 4 * r, v, y[r]);
  }
}

// More rows (or few rows and a K too long for k_q4_stream): the hidden rows come through LDS in
// chunks of four steps, two chunks at a time (straight from k_q4_blocks' image of them), and a
// wave goes through its MT row tiles chunk by chunk, two at a time (a fragment read from LDS
// serves both), their sums in registers. The code of a chunk has no branches between its
// requests, so that each wait is for the oldest alone. Any alignment, any number of groups. PARTS:
// gridDim.y parts of K, their sums to `part`. The sums (b - 16 s) X are MFMAs of the words of scales
// and biases as loaded (by multiply-adds, 64 rows with groups of 32: 220 us instead of 187).
// (V = 151,936, K = 5,120, groups of 64: 16 rows 116 us, 32 rows 129, 64 rows 158, groups of 128:
// 139. Few rows are bound by the weights' loads, as k_q4_stream's, 64 by vector instructions and
// MFMA of two waves a SIMD.)
constexpr int QC_NW = 8;

template <int I>
struct QInt {
  static constexpr int value = I;
};

template <int G, int NT, int MT, bool PARTS>
__global__ __launch_bounds__(QC_NW* WAVE, 2) void k_q4_chunk(const Q4Args a) {
  constexpr int GPS = 128 / G, MPG = 4 / GPS, NS = q4_chunk_sums<G>();
  constexpr int CHUNK = (16 + NS) * NT * 1024;
  constexpr int SW = G == 128 ? 2 : 4;  // words of scales a lane loads
  extern __shared__ __attribute__((aligned(1024))) uint8_t s_all[];
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)s_all;
  const int lane = threadIdx.x & (WAVE - 1), wv = wave_id(), h = lane >> 4, r16 = lane & 15;
  const int nw = blockDim.x / WAVE;
  const int units = (a.w.K + 511) / 512, groups = a.w.K / G, pieces = a.w.K / 32;
  const int v0 = (blockIdx.x * nw + wv) * MT * 16;
  int first = 0, last = units;  // this workgroup's chunks of K
  if constexpr (PARTS) {
    first = (int)((int64_t)units * blockIdx.y / gridDim.y);
    last = (int)((int64_t)units * (blockIdx.y + 1) / gridDim.y);
  }
  const bool sym = a.w.biases == nullptr;
  const uint16_t* side = (h & 1) && !sym ? a.w.biases : a.w.scales;
  const int sofs = G == 32 ? 8 * (h >> 1) : 0;  // the upper quarters: a unit's second eight

  // Two units of weights, the tiles 2 i and 2 i + 1 of a chunk (and the last alone where MT is
  // odd); each part of one is requested anew, for the tile that has the place next, as soon as
  // it has been taken up.
  struct Unit {
    qu32x4 w[4];
    uint32_t s[SW];
  } buf[2];
  // scales are loaded in whole vectors that end inside the row
  auto back_of = [&](int c) { return max(0, c * 4 * GPS + sofs + 2 * SW - groups); };
  auto load_words = [&](Unit& u, int c, int mt, int p) {
    const int v = min(v0 + 16 * mt + r16, a.w.V - 1);
    u.w[p] = *(const qu32x4*)(a.w.words + (int64_t)v * a.w.words_stride +
                              4 * min(16 * min(c, units - 1) + 4 * p + h, pieces - 1));
  };
  auto load_scales = [&](Unit& u, int c, int mt) {
    c = min(c, units - 1);
    const int v = min(v0 + 16 * mt + r16, a.w.V - 1);
    const uint16_t* sp = side + (int64_t)v * a.w.scales_stride + c * 4 * GPS + sofs - back_of(c);
    if constexpr (SW == 2) {
      const qu32x2u q = *(const qu32x2u*)sp;
      u.s[0] = q[0], u.s[1] = q[1];
    } else {
      const qu32x4u q = *(const qu32x4u*)sp;
      u.s[0] = q[0], u.s[1] = q[1], u.s[2] = q[2], u.s[3] = q[3];
    }
  };
  // the hidden rows' chunk c into half c & 1: piece i of nw waves' CHUNK / 1024
  const int share = (CHUNK / 1024 + nw - 1) / nw;
  auto bring = [&](int c) {
    c = min(c, units - 1);
    const uint8_t* from = a.blocks + (int64_t)c * CHUNK + lane * 16;
    for (int i = 0; i < share; ++i) {
      const int e = min(wv * share + i, CHUNK / 1024 - 1) * 1024;
      q4_load_lds<false>(lds + (c & 1) * CHUNK + e, from + e);
    }
  };

  const Q4Masks masks;
  qf32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[i][nt] = qf32x4{0.f, 0.f, 0.f, 0.f};

  // tiles mt .. mt + CNT - 1 of chunk c; the places' next tiles are those of tile mt + 2, + 3,
  // or of the next chunk
  auto compute = [&](int c, auto mt_, auto cnt_) {
    constexpr int M0 = decltype(mt_)::value, CNT = decltype(cnt_)::value;
    uint32_t sw[CNT][2 * GPS];  // the units' scales, in every quarter
    const int back = back_of(c);
    const uint8_t* xc = s_all + (c & 1) * CHUNK + lane * 16;
#pragma unroll
    for (int j = 0; j < CNT; ++j) {
      Unit& u = buf[j];
      // the scales moved back for want of room move into place
#pragma unroll
      for (int d = SW / 2; d > 0; d /= 2)  // by d words
#pragma unroll
        for (int e = 0; e < SW; ++e) u.s[e] = back & (2 * d) ? (e + d < SW ? u.s[e + d] : 0u) : u.s[e];
#pragma unroll
      for (int e = 0; e < SW; ++e) {
        const uint32_t half = (u.s[e] >> 16) | (e + 1 < SW ? u.s[e + 1] << 16 : 0u);
        u.s[e] = back >= 2 * SW ? 0u : back & 1 ? half : u.s[e];
      }
      // sum of (b - 16 s) X over the chunk's groups
      const qu32x4 sb = {u.s[0], u.s[1], SW == 2 ? u.s[0] : u.s[SW - 2], SW == 2 ? u.s[1] : u.s[SW - 1]};
#pragma unroll
      for (int q = 0; q < NS; ++q)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const qu32x4 y = *(const qu32x4*)(xc + ((16 + q) * NT + nt) * 1024);
          acc[M0 + j][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(qbf16x8, y), __builtin_bit_cast(qbf16x8, sb), acc[M0 + j][nt], 0, 0, 0);
        }
#pragma unroll
      for (int e = 0; e < SW; ++e) {
        uint32_t s0 = u.s[e], other = u.s[e];
        q4_swap16(s0, other);
        if constexpr (G == 32) {
          uint32_t s1 = s0;
          q4_swap32(s0, s1);
          sw[j][4 + e] = s1;
        }
        sw[j][e] = s0;
      }
      load_scales(u, M0 + 2 + j < MT ? c : c + 1, M0 + 2 + j < MT ? M0 + 2 + j : j);
    }
    uint32_t w[CNT][4];
#pragma unroll
    for (int i = 0; i < 4 * GPS; ++i) {  // the chunk's groups
      const int p = i / GPS, g = i % GPS;
      if (g == 0) {
#pragma unroll
        for (int j = 0; j < CNT; ++j) {
          q4_order<G>(buf[j].w[p], w[j]);
          load_words(buf[j], M0 + 2 + j < MT ? c : c + 1, M0 + 2 + j < MT ? M0 + 2 + j : j, p);
        }
      }
      qbf16x8 codes[CNT][MPG];
      float sc[CNT];
#pragma unroll
      for (int j = 0; j < CNT; ++j) {
#pragma unroll
        for (int q = 0; q < MPG; ++q) codes[j][q] = q4_codes(w[j][g * MPG + q], masks);
        sc[j] = __uint_as_float(i & 1 ? sw[j][i / 2] & 0xFFFF0000u : sw[j][i / 2] << 16);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        qf32x4 t[CNT];
#pragma unroll
        for (int q = 0; q < MPG; ++q) {
          const qu32x4 x = *(const qu32x4*)(xc + ((4 * p + g * MPG + q) * NT + nt) * 1024);
#pragma unroll
          for (int j = 0; j < CNT; ++j) {
            if (q == 0) t[j] = qf32x4{0.f, 0.f, 0.f, 0.f};
            t[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(qbf16x8, x), codes[j][q], t[j], 0, 0, 0);
          }
        }
#pragma unroll
        for (int j = 0; j < CNT; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[M0 + j][nt][r] = __builtin_fmaf(sc[j], t[j][r], acc[M0 + j][nt][r]);
      }
    }
    // (more than 16 rows: two pairs of tiles at once are more than the registers hold)
    if constexpr (NT > 1) __builtin_amdgcn_sched_barrier(0);
  };
  bring(first);
#pragma unroll
  for (int j = 0; j < (MT > 1 ? 2 : 1); ++j) {
    load_scales(buf[j], first, j);
#pragma unroll
    for (int p = 0; p < 4; ++p) load_words(buf[j], first, j, p);
  }
  for (int c = first; c < last; ++c) {
    // every wave's part of the chunk has arrived (a unit's request is four loads or more, and one
    // or more units were requested since), and none reads the other half any more
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(MT > 1 ? 8 : 4) : "memory");
    if (c + 1 < last) bring(c + 1);
    if constexpr (MT > 1) compute(c, QInt<0>{}, QInt<2>{});
    if constexpr (MT > 3) compute(c, QInt<2>{}, QInt<2>{});
    if constexpr (MT % 2) compute(c, QInt<MT - 1>{}, QInt<1>{});
  }
  // lane: weight row r16, places 4 h + r of each batch tile
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int v = v0 + 16 * i + r16;
    if (v >= a.w.V) continue;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int b = 16 * nt + q4_row(4 * h + r);
        if (b >= a.B) continue;
        if (!PARTS) q4_store(a, b, v, acc[i][nt][r]);
        else a.part[((int64_t)blockIdx.y * a.B + b) * a.w.V + v] = acc[i][nt][r];
      }
  }
}

// The results of a product split along K: its parts' sums, in their order.
__global__ __launch_bounds__(256) void k_q4_join(const Q4Args a, int splits) {
  const int v = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
  if (v >= a.w.V) return;
  float y = 0.0f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) y += a.part[((int64_t)s * a.B + b) * a.w.V + v];
  q4_store(a, b, v, y);
}

// K of fewer than eight groups: one wave a row tile, straightforwardly.
template <int G, int NT>
__global__ __launch_bounds__(WAVE) void k_q4_short(const Q4Args a) {
  constexpr int GPS = 128 / G, MPG = 4 / GPS, CHUNK = (16 + q4_chunk_sums<G>()) * NT * 1024;
  const int lane = threadIdx.x, h = lane >> 4, r16 = lane & 15;
  const int steps = (a.w.K + 127) / 128, groups = a.w.K / G, pieces = a.w.K / 32;
  const int row = blockIdx.x * 16 + r16, v = min(row, a.w.V - 1);
  const uint32_t* wp = a.w.words + (int64_t)v * a.w.words_stride;
  const uint16_t* sp = a.w.scales + (int64_t)v * a.w.scales_stride;
  const uint16_t* bp = a.w.biases ? a.w.biases + (int64_t)v * a.w.scales_stride : nullptr;
  const Q4Masks masks;
  qf32x4 acc[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) acc[nt] = qf32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < steps; ++s) {
    const uint8_t* xc = a.blocks + (int64_t)(s >> 2) * CHUNK + (s & 3) * 4 * NT * 1024 + lane * 16;
    uint32_t w[4];
    q4_order<G>(*(const qu32x4*)(wp + 4 * min(4 * s + h, pieces - 1)), w);
#pragma unroll
    for (int g = 0; g < GPS; ++g) {
      const int gi = s * GPS + g;
      if (gi >= groups) break;
      const float sc = __uint_as_float((uint32_t)sp[gi] << 16);
      const float bi = bp ? __uint_as_float((uint32_t)bp[gi] << 16) : -8.0f * sc;
      const float off = bi - 16.0f * sc;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        qf32x4 t = {0.f, 0.f, 0.f, 0.f}, xs = t;
#pragma unroll
        for (int q = 0; q < MPG; ++q) {
          const int m = g * MPG + q;
          const qu32x4 x = *(const qu32x4*)(xc + (m * NT + nt) * 1024);
          xs = q4_sum(x, xs);
          t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(qbf16x8, x), q4_codes(w[m], masks), t, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[nt][r] = __builtin_fmaf(sc, t[r], __builtin_fmaf(off, xs[r], acc[nt][r]));
      }
    }
  }
  if (row >= a.w.V) return;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int b = 16 * nt + q4_row(4 * h + r);
      if (b < a.B) q4_store(a, b, row, acc[nt][r]);
    }
}

// ---- host ---------------------------------------------------------------------------------
static int q4_tiles_n(int B) { return B <= 16 ? 1 : B <= 32 ? 2 : 4; }

static int64_t q4_blocks_bytes(int B, int K) {
  return ((int64_t)K + 511) / 512 * (16 + 3) * q4_tiles_n(B) * 1024;
}

// k_q4_chunk's row tiles, over all its parts of K, are this many at most: eight waves a CU.
constexpr int QC_SPLIT = 2048;

// None where k_q4_stream (or k_q4_dma) takes the rows whatever the groups: they fit its LDS.
int64_t q4_workspace(int B, int K) {
  const int64_t steps = ((int64_t)K + 511) / 512 * 4;
  const bool one = B <= 4 && steps * q4_step_bytes<32, 1>() + QS_NW * 2 * 1 * WAVE * 4 <= (int64_t)QS_LDS;
  const bool two = B <= 8 && steps * q4_step_bytes<32, 2>() + QS_NW * 2 * 2 * WAVE * 4 <= (int64_t)QS_LDS;
  if (K >= 8 * 128 && (one || two)) return 0;
  const int rows = B < 64 ? B : 64;
  return q4_blocks_bytes(B, K) + (int64_t)QC_SPLIT * 16 * rows * 4;
}

// A launch with more than 64 KB of LDS, which a kernel has to be told of once on each device. (One
// that cannot be told is not launched; the call ends with that error.)
template <auto KERNEL, class... More>
static bool q4_big_lds(dim3 grid, size_t lds, hipStream_t st, const Q4Args& a, int waves, More... more) {
  static std::atomic<uint64_t> told{0};  // a bit a device
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess) return true;
  const uint64_t bit = (uint64_t)1 << (device & 63);
  if (!(told.load(std::memory_order_relaxed) & bit)) {
    if (hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize,
                            (int)QS_LDS) != hipSuccess)
      return true;
    told.fetch_or(bit, std::memory_order_relaxed);
  }
  hipLaunchKernelGGL(KERNEL, grid, dim3(waves * WAVE), lds, st, a, more...);
  return true;
}

template <int G, int RB, int D>
static bool q4_stream(const Q4Args& a, hipStream_t st) {
  const int steps = (a.w.K + 511) / 512 * 4, tiles = (a.w.V + 15) / 16;
  const size_t own = (size_t)steps * q4_step_bytes<G, RB>();
  // Through LDS with seven waves or more, where each lane's scale load may be two groups by two:
  // at V = 65,536, groups of 64, 8 rows, K = 5,120 (seven waves) 48.1 us, through registers 50.8;
  // K = 6,656 (five) 67.1 against 60.2, K = 8,192 (two) 139 against 76.
  const bool even = (a.w.K / G) % 2 == 0 && a.w.scales_stride % 2 == 0 && ((uintptr_t)a.w.scales & 3) == 0 &&
                    ((uintptr_t)a.w.biases & 3) == 0 && a.w.K >= 8 * G;
  const int nw = own < QS_LDS ? (int)((QS_LDS - own) / 10240) : 0;
  if (even && nw >= 7) {
    const dim3 grid((unsigned)(tiles < 256 ? tiles : 256));
    const int w = nw < QS_NW ? nw : QS_NW;
    const size_t lds = own + (size_t)w * 10240;
    return a.w.K % 512 == 0 ? q4_big_lds<k_q4_dma<G, RB, true>>(grid, lds, st, a, w, tiles)
                            : q4_big_lds<k_q4_dma<G, RB, false>>(grid, lds, st, a, w, tiles);
  }
  const size_t lds = (size_t)steps * q4_step_bytes<G, RB>() + (size_t)QS_NW * 2 * RB * WAVE * 4;
  if (lds > QS_LDS || a.w.K < 8 * G) return false;
  const dim3 grid((unsigned)(tiles < 256 ? tiles : 256));
  return a.w.K % 512 == 0 ? q4_big_lds<k_q4_stream<G, RB, D, true>>(grid, lds, st, a, QS_NW, tiles)
                          : q4_big_lds<k_q4_stream<G, RB, D, false>>(grid, lds, st, a, QS_NW, tiles);
}

template <int G, int NT, int MT, bool PARTS = false>
static void q4_chunk(const Q4Args& a, int nw, int splits, hipStream_t st) {
  const int tiles = (a.w.V + 15) / 16, each = nw * MT;
  q4_big_lds<k_q4_chunk<G, NT, MT, PARTS>>(dim3((unsigned)((tiles + each - 1) / each), (unsigned)splits),
                                    (size_t)2 * (16 + q4_chunk_sums<G>()) * NT * 1024, st, a, nw);
}

template <int G, int NT>
static void q4_blocks(const Q4Args& a, hipStream_t st) {
  const int tiles = (a.w.V + 15) / 16;
  hipLaunchKernelGGL((k_q4_blocks<G, NT>), dim3((unsigned)((a.w.K + 511) / 512), NT), dim3(4 * WAVE), 0, st, a);
  if (a.w.K < 8 * G) {
    hipLaunchKernelGGL((k_q4_short<G, NT>), dim3((unsigned)tiles), dim3(WAVE), 0, st, a);
    return;
  }
  // Less than a round of row tiles: K is split over workgroups and the parts' sums joined, where
  // that saves more chunks (about `alone` us each, `full` with eight waves) than the join costs;
  // then the fewest waves a workgroup that fill the CUs. (K = 5,120, groups of 64, split and not:
  // 16 rows, V = 4,096 13.3 and 20.3 us, V = 16,000 22.9 and 26.2; 64 rows, V = 4,096 20.9 and
  // 39.5, V = 16,000 33.7 and 39.6; 16 rows, K = 1,024, V = 8,192 13.6 and 12.3. Without a split,
  // 16 rows, V = 4,096, eight waves: 24.0.)
  if (tiles < QC_SPLIT) {
    const int units = (a.w.K + 511) / 512;
    const double alone = NT == 1 ? 1.7 : NT == 2 ? 2.2 : 3.5, full = NT == 1 ? 2.5 : NT == 2 ? 3.2 : 5.0;
    int splits = QC_SPLIT / tiles < units ? QC_SPLIT / tiles : units;
    if ((units + splits - 1) / splits * full + 3.0 > units * alone) splits = 1;
    int nw = QC_NW;
    while (nw > 2 && (tiles + nw / 2 - 1) / (nw / 2) * splits <= 256) nw /= 2;
    if (splits == 1) {
      q4_chunk<G, NT, 1>(a, nw, 1, st);
      return;
    }
    q4_chunk<G, NT, 1, true>(a, nw, splits, st);
    hipLaunchKernelGGL(k_q4_join, dim3((unsigned)((a.w.V + 255) / 256), (unsigned)a.B), dim3(256), 0, st, a, splits);
    return;
  }
  // Tiles a wave, by the time of its rounds over the CUs (in tiles, as measured; the last round by
  // how full it is). Two tiles read the hidden rows' fragments from LDS once, and more tiles wait
  // fewer times, but a round of five tiles that is half empty takes as long as one of four. (K =
  // 5,120, groups of 64, V = 151,936, one, three and five tiles: 64 rows 220, 192 and 172 us, 32 rows
  // 146, 147 and 131; V = 65,536, 64 rows, one, two and five: 90, 77 and 125; 32 rows, one and five:
  // 65 and 105. 16 rows, with four workgroups a CU: V = 151,936 115 us by one tile, 128 by five.)
  int best = 1;
  if constexpr (NT > 1) {
    const double round[6] = {0.0, 1.35, 2.28, 3.2, 4.0, 5.0}, all = (double)tiles / (256 * QC_NW);
    double least = NT == 2 ? 0.3 + 1.11 * all : 1e30;  // (32 rows, one tile: two workgroups a CU)
    for (int mt = NT == 2 ? 3 : 1; mt <= 5; ++mt) {
      const double n = all / mt, whole = (double)(int64_t)n;
      const double cost = round[mt] * (n == whole ? n : whole + 0.75 + 0.25 * (n - whole));
      if (cost < least) least = cost, best = mt;
    }
  }
  if (best == 1) q4_chunk<G, NT, 1>(a, QC_NW, 1, st);
  if constexpr (NT > 2)
    if (best == 2) q4_chunk<G, NT, 2>(a, QC_NW, 1, st);
  if constexpr (NT > 1) {
    if (best == 3) q4_chunk<G, NT, 3>(a, QC_NW, 1, st);
    if (best == 4) q4_chunk<G, NT, 4>(a, QC_NW, 1, st);
    if (best == 5) q4_chunk<G, NT, 5>(a, QC_NW, 1, st);
  }
}

// Up to 8 rows from LDS (V = 151,936, K = 5,120, groups of 64, 8 rows: 99 us, by k_q4_chunk 116; V =
// 8,192: 12.7 against 21.4), up to 4 of them with half the places (4 rows: 92.8 us, as up to 8: 95.6).
template <int G>
static void q4_logits(const Q4Args& a, hipStream_t st) {
  if (a.B <= 4 && q4_stream<G, 1, 2>(a, st)) return;
  if (a.B <= 8 && q4_stream<G, 2, 2>(a, st)) return;
  const int nt = q4_tiles_n(a.B);
  if (nt == 1) q4_blocks<G, 1>(a, st);
  else if (nt == 2) q4_blocks<G, 2>(a, st);
  else q4_blocks<G, 4>(a, st);
}

hipError_t launch_q4_logits(const void* x, int64_t x_stride, int B, int K, const uint32_t* words,
                            int64_t words_stride, const uint16_t* scales, const uint16_t* biases,
                            int64_t scales_stride, int group, int V, void* workspace, void* out,
                            bool out_f32, int64_t out_stride, hipStream_t st) {
  for (int64_t b = 0; b < B; b += 64) {  // the weights are read once per 64 rows
    Q4Args a{};
    a.w = Q4Weights{words, words_stride, scales, biases, scales_stride, V, K};
    a.x = (const uint16_t*)x + b * x_stride;
    a.x_stride = x_stride;
    a.B = B - b < 64 ? (int)(B - b) : 64;
    a.blocks = (uint8_t*)workspace;
    a.part = (float*)(a.blocks + q4_blocks_bytes(B < 64 ? B : 64, K));
    a.out = (uint8_t*)out + b * out_stride * (out_f32 ? 4 : 2);
    a.out_stride = out_stride;
    a.out_f32 = out_f32;
    if (group == 32) q4_logits<32>(a, st);
    else if (group == 64) q4_logits<64>(a, st);
    else q4_logits<128>(a, st);
  }
  return hipGetLastError();
}

hipError_t launch_q4_pack(const void* w, bool f32, int64_t w_stride, int V, int K, int group,
                          uint32_t* words, uint16_t* scales, uint16_t* biases, hipStream_t st) {
  const Q4Pack a{w, w_stride, V, K, words, scales, biases};
  const int64_t blocks = ((int64_t)V * (K / 8) + 255) / 256;
  const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192));
#define STRIM_PACK(G_, F_, S_) hipLaunchKernelGGL((k_q4_pack<G_, F_, S_>), grid, dim3(256), 0, st, a)
#define STRIM_PACK_G(F_, S_)                \
  do {                                      \
    if (group == 32) STRIM_PACK(32, F_, S_); \
    else if (group == 64) STRIM_PACK(64, F_, S_); \
    else STRIM_PACK(128, F_, S_);           \
  } while (0)
  if (f32 && biases) STRIM_PACK_G(true, false);
  else if (f32) STRIM_PACK_G(true, true);
  else if (biases) STRIM_PACK_G(false, false);
  else STRIM_PACK_G(false, true);
#undef STRIM_PACK_G
#undef STRIM_PACK
  return hipGetLastError();
}

hipError_t launch_q4_unpack(const uint32_t* words, int64_t words_stride, const uint16_t* scales,
                            const uint16_t* biases, int64_t scales_stride, int group, int V, int K,
                            void* out, bool out_f32, int64_t out_stride, hipStream_t st) {
  const Q4Weights a{words, words_stride, scales, biases, scales_stride, V, K};
  const int64_t blocks = ((int64_t)V * (K / (out_f32 ? 4 : 8)) + 255) / 256;
  const int64_t most = out_f32 ? 2048 : 8192;
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
#define STRIM_UNPACK(G_)                                                                          \
  do {                                                                                            \
    if (out_f32) hipLaunchKernelGGL((k_q4_unpack<G_, true>), grid, dim3(256), 0, st, a, out, out_stride); \
    else hipLaunchKernelGGL((k_q4_unpack<G_, false>), grid, dim3(256), 0, st, a, out, out_stride); \
  } while (0)
  if (group == 32) STRIM_UNPACK(32);
  else if (group == 64) STRIM_UNPACK(64);
  else STRIM_UNPACK(128);
#undef STRIM_UNPACK
  return hipGetLastError();
}

}  // namespace strim
