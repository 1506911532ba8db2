// loss_kernels.hip — cross entropy of the vocabulary projection's logits, without keeping the
// logits, and its gradients, for bf16 hidden states [N, K] and a bf16 lm_head [V, K].
//
//   x[n][v] = sum_k hidden[n][k] lm_head[v][k]          (float32 accumulation)
//   lse[n]  = log sum_v exp(x[n][v]),  loss[n] = lse[n] - x[n][target[n]]
//   p[n][v] = (g[n] + z[n]) exp(x[n][v] - lse[n]) - g[n] [v = target[n]]
//   d_hidden[n][k]  = sum_v p[n][v] lm_head[v][k]
//   d_lm_head[v][k] = sum_n p[n][v] hidden[n][k]
// with g = dL/dloss and z = dL/dlse.
//
// Four products of 2 N V K operations: the logits twice (once for their row statistics, once
// more for p), and one for each gradient. What is kept between them is a (max, sum) pair per
// row and slice of the vocabulary (the 32, 64 or 128 of its rows that one wave has), and p of one
// piece of the vocabulary, rounded to bf16 for the two gradient products (the gradients are bf16
// themselves; their sums are float32).
//
// k_loss_gemm is all four: a tile of C = A B^T on v_mfma_f32_16x16x32_bf16, its operands
// brought by 16-byte loads straight into LDS, one stage of 64 along the reduction ahead of
// the multiplies. An operand whose rows run along the reduction is read from LDS 8 elements
// a lane; one whose rows run across it (both of d_lm_head's, the projection in d_hidden) is
// transposed on its way from LDS to the registers (ds_read_b64_tr_b16), so nothing is laid
// out anew in memory.
#include "kernels.hpp"

namespace strim {

typedef __bf16 lbf16x8 __attribute__((ext_vector_type(8)));
typedef float lf32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t lu32x4 __attribute__((ext_vector_type(4)));
typedef short ls16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) ls16x4 lds_s16x4;
typedef __attribute__((address_space(3))) lu32x4 lds_u32x4;

constexpr int LG_BK = 64;                 // reduction elements a stage
constexpr uint32_t LG_RANGE = 0x40000000u;  // bytes a buffer descriptor spans; a lane that has
                                            // nothing to load points past it and gets zeros

enum LossMode { LM_STATS = 0, LM_PROB = 1, LM_DHID = 2, LM_DHEAD = 3 };

// One operand: `rows` valid rows (of the tile dimension) from `p`, `red` valid elements along
// the reduction. TR false: element (row, k) at p[row stride + k]; true: p[k stride + row].
struct LossOperand {
  const uint16_t* p;
  int64_t stride;
  int32_t rows;
};

struct LossGemm {
  LossOperand a, b;        // a: the tile's M side, b: its N side
  int32_t red;             // reduction length
  int32_t split_red;       // reduction elements a split (a multiple of LG_BK)
  int32_t tiles_m, tiles_n, splits;
  // LM_STATS, LM_PROB: M = vocabulary rows from v0, N = tokens
  int32_t v0, ignore_index;
  int32_t V;
  const int32_t* targets;
  float2* part;            // LM_STATS [slice][N]: max, sum exp(x - max) of a vocabulary slice
  float* tlogit;           // LM_STATS [N]: the target's logit
  const float *lse, *grad_loss, *grad_lse;
  float* scale;            // what p was divided by: LM_PROB writes it, the gradients read it
  uint16_t* out16;         // LM_PROB p [N][out_stride]; LM_DHEAD [v][out_stride]
  int64_t out_stride;
  float* out32;            // LM_DHID [split][N][out_stride]
  int32_t accumulate;      // LM_DHID: add to what out32 holds
};

typedef float lf32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 lbf16x2 __attribute__((ext_vector_type(2)));

// Two floats rounded to nearest even, as one word (NaN stays NaN).
__device__ __forceinline__ uint32_t loss_pack2(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(lf32x2{lo, hi}, lbf16x2));
}
__device__ __forceinline__ uint2 loss_pack4(const float* f) {
  return make_uint2(loss_pack2(f[0], f[1]), loss_pack2(f[2], f[3]));
}

// Words of two neighbouring 16 x 16 tiles, four rows (two words) a lane each, exchanged so that
// a lane has eight rows of one of them: even quarters of the wave the first tile's rows 8 (h / 2)
// .. + 7, odd ones the second's.
__device__ __forceinline__ uint4 loss_join8(uint2 a, uint2 b) {
  const auto x = __builtin_amdgcn_permlane16_swap(a.x, b.x, false, false);
  const auto y = __builtin_amdgcn_permlane16_swap(a.y, b.y, false, false);
  return make_uint4(x[0], y[0], x[1], y[1]);
}

__device__ __forceinline__ float loss_exp(float x) {
  return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f);
}

// 64 lanes' 16 bytes each, to LDS from `dst` (the same in every lane) in lane order.
__device__ __forceinline__ void loss_load_lds(uint32_t dst, uint32_t voff, lu32x4 rsrc) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               ::"s"(dst), "v"(voff), "s"(rsrc) : "memory");
}

// The part of an operand's stage that one wave loads, and its fragments' places in LDS.
// A stage holds, TR false, ROWS rows of 64 elements (128 bytes, 16-byte piece c at place
// c ^ (row & 7)); TR true, 64 rows of ROWS elements (32-byte piece c at place c ^ f(row)):
// with these orders the lanes of one LDS read meet all banks evenly.
template <bool TR, int ROWS, int NW>
struct LossTile {
  static constexpr int BYTES = ROWS * 2 * LG_BK;
  static constexpr int NI = BYTES / 1024 / NW;         // load instructions a wave
  static constexpr int RPI = TR ? 512 / ROWS : 8;      // rows an instruction covers
  static constexpr int LPR = 64 / RPI;                 // lanes a row
  static_assert(NI >= 1 && NI * NW * 1024 == BYTES, "whole instructions");
  uint32_t voff[NI];
  int kofs;
  const uint16_t* base;
  int64_t step;
  uint32_t lds0;

  static __device__ __forceinline__ int f(int row) { return (row & 3) | ((row >> 1) & 4); }

  __device__ __forceinline__ void init(const LossOperand& o, int row0, int red0, int wv, int lane) {
    const int r0 = wv * NI * RPI + lane / LPR;
    if constexpr (TR) {
      base = o.p + (int64_t)red0 * o.stride + row0;
      step = (int64_t)LG_BK * o.stride;
      kofs = r0;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int r = r0 + j * RPI, c = lane % LPR;
        const int col = (((c >> 1) ^ f(r)) << 4) + ((c & 1) << 3);
        voff[j] = row0 + col < o.rows ? (uint32_t)(2 * (r * (int)o.stride + col)) : LG_RANGE;
      }
    } else {
      base = o.p + (int64_t)row0 * o.stride + red0;
      step = LG_BK;
      const int c = (lane & 7) ^ (lane >> 3);
      kofs = 8 * c;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int r = r0 + j * RPI;
        voff[j] = row0 + r < o.rows ? (uint32_t)(2 * (r * (int)o.stride + 8 * c)) : LG_RANGE;
      }
    }
    lds0 = (uint32_t)(wv * NI * 1024);
  }

  // requests stage `s` (elements s * 64 onwards of a reduction of `red`) into LDS at `lds`
  __device__ __forceinline__ void load(uint32_t lds, int s, int red) const {
    const uint64_t at = (uint64_t)(base + (int64_t)s * step);
    lu32x4 rsrc;
    rsrc[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)at);
    rsrc[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32) & 0xFFFF);
    rsrc[2] = LG_RANGE;
    rsrc[3] = 0x00020000u;
    const int left = red - s * LG_BK - kofs;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const bool in = left > (TR ? j * RPI : 0);
      loss_load_lds(__builtin_amdgcn_readfirstlane((int)(lds + lds0 + j * 1024)),
                    in ? voff[j] : LG_RANGE, rsrc);
    }
  }
};

// Fragment reads: lane l holds elements 8 (l / 16) .. + 7 along the reduction of row l % 16
// of the 16-row tile t0 + i, half kk (32 of the stage's 64 elements).
template <bool TR, int ROWS>
struct LossFrag {
  uint32_t at0, at1;  // TR: at0 the row part, at1 the piece's xor
  __device__ __forceinline__ void init(int t0, int lane) {
    const int h = lane >> 4, j = lane & 15;
    if constexpr (TR) {
      at0 = (uint32_t)((8 * h + (j >> 2)) * (2 * ROWS) + 8 * (j & 3));
      at1 = (uint32_t)(t0 * 32) ^ (uint32_t)(((j >> 2) | ((h & 1) << 2)) * 32);
    } else {
      at0 = (uint32_t)((t0 * 16 + j) * 128 + ((h ^ (j & 7)) << 4));
      at1 = at0 ^ 64u;
    }
  }
  __device__ __forceinline__ lbf16x8 get(uint32_t lds, int i, int kk) const {
    if constexpr (TR) {
      const uint32_t a = lds + at0 + (at1 ^ (uint32_t)(i * 32)) + (uint32_t)(kk * 32 * 2 * ROWS);
      const ls16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)a);
      const ls16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(a + 4 * 2 * ROWS));
      return __builtin_bit_cast(lbf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const uint32_t a = lds + (kk ? at1 : at0) + (uint32_t)(i * 2048);
      return __builtin_bit_cast(lbf16x8, *(const lds_u32x4*)(uintptr_t)a);
    }
  }
};

// Workgroup -> tile: each XCD (workgroups are dealt to the eight in turn) takes a run of
// neighbouring tiles, eight of the N side by as many of the M side as are in flight, so that
// its L2 serves each operand slab to several workgroups.
__device__ __forceinline__ void loss_tile(int tiles_m, int tiles_n, int splits, int& tm, int& tn,
                                          int& split) {
  const int tiles = tiles_m * tiles_n, total = tiles * splits, b = blockIdx.x;
  const int x = b & 7, per = total >> 3, rem = total & 7;
  int id = x * per + min(x, rem) + (b >> 3);
  split = id / tiles;
  id -= split * tiles;
  const int g = id / (8 * tiles_m), r = id - g * 8 * tiles_m;
  const int wide = min(8, tiles_n - 8 * g);
  tn = 8 * g + r % wide;
  tm = r / wide;
}

// The number that p is held divided by: the first nonzero gradient of a row that counts, among
// the first 1,024 (ordinary sizes only; else 1). Where every row weighs the same, as in a mean,
// p then holds exp(x - lse) - [v = t] itself, whose -1 is exact. With the weight in it every
// target's -g would be rounded alike, an error that no sum averages out: N = 2,000 rows at
// weights of 1/1,600 gave d_lm_head 1.5 times the relative error of a float32 evaluation rounded
// once, and 1.2 times without.
__device__ __forceinline__ float loss_scale(const LossGemm& g, int lane) {
  for (int n0 = 0; n0 < min(g.b.rows, 1024); n0 += WAVE) {
    const int n = min(n0 + lane, g.b.rows - 1), t = g.targets[n];
    const float gl = g.grad_loss[n], gz = g.grad_lse ? g.grad_lse[n] : 0.0f;
    const float c = t == g.ignore_index || t < 0 || t >= g.V ? 0.0f : gl != 0.0f ? gl : gz;
    const uint64_t have = __ballot(fabsf(c) > 1e-12f && fabsf(c) < 1e12f);
    if (have) return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(c), __builtin_ctzll(have)));
  }
  return 1.0f;
}

// What LM_PROB needs of a token.
struct LossRow {
  float lse, top, gl;  // p = top exp(x - lse) - gl [v = target]
  int32_t target;      // INT_MIN: the row counts for nothing
};

// WM x WN waves of TM x TN tiles of 16 x 16; R stages in LDS.
template <int MODE, int WM, int WN, int TM, int TN, int R>
__global__ __launch_bounds__(WM* WN* WAVE, 2) void k_loss_gemm(const LossGemm g) {
  constexpr bool ATR = MODE == LM_DHID || MODE == LM_DHEAD, BTR = MODE == LM_DHEAD;
  constexpr int NW = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16;
  typedef LossTile<ATR, BM, NW> TileA;
  typedef LossTile<BTR, BN, NW> TileB;
  constexpr int STAGE = TileA::BYTES + TileB::BYTES, LOADS = TileA::NI + TileB::NI;
  __shared__ __attribute__((aligned(1024))) uint8_t s_buf[R * STAGE];
  const uint32_t lds = (uint32_t)(uintptr_t)(lds_u8*)s_buf;
  const int lane = threadIdx.x & (WAVE - 1), wv = wave_id();
  const int wm = wv / WN, wn = wv % WN;
  int tm, tn, split;
  loss_tile(g.tiles_m, g.tiles_n, g.splits, tm, tn, split);
  const int red0 = split * g.split_red, red = max(0, min(g.split_red, g.red - red0));
  const int steps = (red + LG_BK - 1) / LG_BK;
  TileA ta;
  TileB tb;
  ta.init(g.a, tm * BM, red0, wv, lane);
  tb.init(g.b, tn * BN, red0, wv, lane);
  auto request = [&](uint32_t at, int s) {
    ta.load(at, s, red);
    tb.load(at + TileA::BYTES, s, red);
  };
  // (past the reduction's end zeros are requested: the count of open requests is fixed)
#pragma unroll
  for (int s = 0; s < R; ++s) request(lds + s * STAGE, s);
  // (here their loads wait with the first stages, after the product they would wait alone: 8 us of
  // every tile)
  __shared__ LossRow s_row[MODE == LM_PROB ? BN : 1];
  if constexpr (MODE == LM_PROB) {
    const float scale = loss_scale(g, lane);
    if (blockIdx.x == 0 && threadIdx.x == 0) *g.scale = scale;
    for (int c = threadIdx.x; c < BN; c += NW * WAVE) {
      const int n = min(tn * BN + c, g.b.rows - 1), t = g.targets[n];
      const float gl = g.grad_loss[n], gz = g.grad_lse ? g.grad_lse[n] : 0.0f, lse = g.lse[n];
      const bool live = t != g.ignore_index && t >= 0 && t < g.V;
      s_row[c] = live ? LossRow{lse, (gl + gz) / scale, gl / scale, t} : LossRow{0.0f, 0.0f, 0.0f, INT_MIN};
    }
  }
  LossFrag<ATR, BM> fa;
  LossFrag<BTR, BN> fb;
  fa.init(wm * TM, lane);
  fb.init(wn * TN, lane);

  lf32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = lf32x4{0.f, 0.f, 0.f, 0.f};

  // R stages in LDS and two halves (32 of a stage's 64) in registers: while a half is
  // multiplied the next one is read from LDS, so that a stage's first half is read, and the
  // barrier that says it has arrived passed, before the multiplies of the stage before it are
  // over. The stage R after one is requested into the place that this barrier frees.
  lbf16x8 af[2][TM], bf[2][TN];
  auto frags = [&](uint32_t at, int kk) {
#pragma unroll
    for (int j = 0; j < TN; ++j) bf[kk][j] = fb.get(at + TileA::BYTES, j, kk);
#pragma unroll
    for (int i = 0; i < TM; ++i) af[kk][i] = fa.get(at, i, kk);
  };
  auto multiply = [&](int kk) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[kk][i], bf[kk][j], acc[i][j], 0, 0, 0);
  };
  // one LDS read to every few multiplies
  auto interleave = [&]() {
    constexpr int READS = TM * (ATR ? 2 : 1) + TN * (BTR ? 2 : 1), MUL = TM * TN;
    constexpr int EACH = MUL / READS > 0 ? MUL / READS : 1;
#pragma unroll
    for (int i = 0; i < READS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, MUL, 0);
  };
  uint32_t cur = lds;
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((R - 1) * LOADS) : "memory");
  frags(cur, 0);
  for (int s = 0; s < steps; ++s) {
    const uint32_t nxt = cur == lds + (R - 1) * STAGE ? lds : cur + STAGE;
    frags(cur, 1);
    multiply(0);
    interleave();
    // the next stage has arrived, and every wave has read this one
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((R - 2) * LOADS) : "memory");
    if (R > 2 || s + R < steps) request(cur, s + R);
    frags(nxt, 0);  // (after the last stage: zeros, unused)
    multiply(1);
    interleave();
    cur = nxt;
  }
  // none left open (of two stages: the second one's, where there was no step)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // lane l holds C[row 4 (l / 16) + r][column l % 16] of each 16 x 16 tile
  const int h = lane >> 4, c16 = lane & 15;
  const int mw = tm * BM + wm * TM * 16, m0 = mw + 4 * h;
  const int n0 = tn * BN + wn * TN * 16 + c16;
  // bf16 results of column `row` (rows of `out` run along the M side): sixteen bytes a lane
  const int mh = mw + 16 * (h & 1) + 8 * (h >> 1);
  auto store = [&](uint16_t* out, int i, uint2 a, uint2 b, int valid) {
    const uint4 q = loss_join8(a, b);
    if (mh + 16 * i < valid) *(uint4*)(out + mh + 16 * i) = q;
  };
  static_assert(TM % 2 == 0, "tiles are stored by twos");
  if constexpr (MODE == LM_STATS || MODE == LM_PROB) {
    // Past the vocabulary: nothing. (p's last columns too: d_hidden's product reads whole 16-byte
    // pieces, and exp(0 - lse) would be infinite there for a row whose lse is below -88.7.)
    const int left = g.V - g.v0;
    if (mw + TM * 16 > left) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (m0 + 16 * i + r >= left)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j][r] = -INFINITY;
    }
  }
  if constexpr (MODE == LM_STATS) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + 16 * j;
      const int t = n < g.b.rows ? g.targets[n] : -1;
      const int at = t >= 0 && t < g.V ? t - g.v0 - m0 : -1;  // the target's place among this lane's rows
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if (at >= 16 * i && at < 16 * i + 4)
          g.tlogit[n] = at == 16 * i ? acc[i][j][0] : at == 16 * i + 1 ? acc[i][j][1]
                        : at == 16 * i + 2 ? acc[i][j][2] : acc[i][j][3];
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[i][j][r]);
      }
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float ref = mx == -INFINITY ? 0.0f : mx;  // a slice of -inf alone adds nothing
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += loss_exp(acc[i][j][r] - ref);
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (h == 0 && n < g.b.rows)
        g.part[(int64_t)(tm * WM + wm) * g.b.rows + n] = make_float2(mx, sum);
    }
  } else if constexpr (MODE == LM_PROB) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + 16 * j;
      const LossRow row = s_row[n - tn * BN];
      const float lse = row.lse, top = row.top, gl = row.gl;
      const uint32_t keep = row.target != INT_MIN ? 0xFFFFFFFFu : 0u;  // whatever a dead row holds
      const int at = row.target != INT_MIN ? row.target - g.v0 - m0 : -1;  // the target among this lane's rows
      uint2 w[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        float p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = top * loss_exp(acc[i][j][r] - lse);
        if (at >= 16 * i && at < 16 * i + 4)
#pragma unroll
          for (int r = 0; r < 4; ++r) p[r] -= at == 16 * i + r ? gl : 0.0f;
        w[i] = loss_pack4(p);
        w[i].x &= keep, w[i].y &= keep;
      }
      // (columns past the vocabulary are inside the row, and zero)
      if (n < g.b.rows)
#pragma unroll
        for (int i = 0; i < TM; i += 2)
          store(g.out16 + (int64_t)n * g.out_stride, i, w[i], w[i + 1], (int)g.out_stride);
    }
  } else if constexpr (MODE == LM_DHID) {
    const float scale = *g.scale;
    float* out = g.out32 + (int64_t)split * g.b.rows * g.out_stride;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + 16 * j;
      if (n >= g.b.rows) continue;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int k = m0 + 16 * i;
        if (k >= g.a.rows) continue;
        lf32x4* at = (lf32x4*)(out + (int64_t)n * g.out_stride + k);
        const lf32x4 y = scale * acc[i][j];
        *at = g.accumulate ? *at + y : y;
      }
    }
  } else {
    const float scale = g.scale ? *g.scale : 1.0f;  // (none without rows)
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int v = n0 + 16 * j;
      uint2 w[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const float f[4] = {scale * acc[i][j][0], scale * acc[i][j][1], scale * acc[i][j][2],
                            scale * acc[i][j][3]};
        w[i] = loss_pack4(f);
      }
      if (v < g.b.rows)
#pragma unroll
        for (int i = 0; i < TM; i += 2)
          store(g.out16 + (int64_t)v * g.out_stride, i, w[i], w[i + 1], g.a.rows);
    }
  }
}

// Merges two (max, sum exp(x - max)) pairs; a max of -inf carries no sum.
__device__ __forceinline__ void loss_merge(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.0f : top;
  s = s * loss_exp(m - ref) + s2 * loss_exp(m2 - ref);
  m = top;
}

// The rows' results from their slices' pairs: TOK tokens a workgroup of 256, the slices of a
// token dealt to 256 / TOK threads in a fixed order.
template <int TOK>
__global__ __launch_bounds__(256) void k_loss_rows(const float2* part, int slices, int N,
                                                   const float* tlogit, const int32_t* targets,
                                                   int ignore_index, int V, float* out_loss,
                                                   float* out_lse, int32_t* out_status) {
  constexpr int W = 256 / TOK;
  __shared__ float2 s_p[W][TOK];
  const int tok = threadIdx.x % TOK, w = threadIdx.x / TOK;
  const int n = blockIdx.x * TOK + tok;
  float m = -INFINITY, s = 0.0f;
  constexpr int U = 8;  // slices requested together
  if (n < N)
    for (int q = w; q < slices; q += U * W) {
      float2 p[U];
#pragma unroll
      for (int u = 0; u < U; ++u) p[u] = part[(int64_t)min(q + u * W, slices - 1) * N + n];
      float top = m;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (q + u * W >= slices) p[u] = make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, p[u].x);
      }
      const float ref = top == -INFINITY ? 0.0f : top;
      s *= loss_exp(m - ref);
#pragma unroll
      for (int u = 0; u < U; ++u) s += p[u].y * loss_exp(p[u].x - ref);
      m = top;
    }
  s_p[w][tok] = make_float2(m, s);
  for (int d = W / 2; d > 0; d >>= 1) {
    __syncthreads();
    if (w < d) {
      const float2 p = s_p[w + d][tok];
      loss_merge(m, s, p.x, p.y);
      s_p[w][tok] = make_float2(m, s);
    }
  }
  if (w != 0 || n >= N) return;
  const int t = targets[n];
  const float ls = logf(s), lse = m + ls;
  const bool known = t >= 0 && t < V, live = known && t != ignore_index;
  // (not from lse, which is rounded to the largest logit's spacing)
  const float loss = live ? (m - tlogit[n]) + ls : 0.0f;
  if (out_lse) out_lse[n] = lse;
  out_loss[n] = loss;
  if (out_status)
    out_status[n] = t == ignore_index ? STRIM_OK
                    : !known          ? STRIM_EINVAL
                    : fabsf(loss) < INFINITY ? STRIM_OK
                                             : STRIM_ENONFINITE;
}

// Hidden rows for the projection's gradient, contiguous: a row without a target is zeroed, so
// that what its padding holds (a NaN too) meets no weight.
__global__ __launch_bounds__(256) void k_loss_rows_in(const uint16_t* x, int64_t stride, int N,
                                                      int K, const int32_t* targets,
                                                      int ignore_index, int V, uint16_t* out) {
  const int n = blockIdx.x;
  const int t = targets[n];
  const bool live = t != ignore_index && t >= 0 && t < V;
  for (int k = 8 * threadIdx.x; k < K; k += 8 * 256) {
    const uint4 q = *(const uint4*)(x + (int64_t)n * stride + k);
    *(uint4*)(out + (int64_t)n * K + k) = live ? q : make_uint4(0, 0, 0, 0);
  }
}

// d_hidden from the splits' sums, added in order and rounded once; eight are requested together (one
// row, K = 1,024: 6.0 us, one after the other 18.0, sixteen 7.6).
__global__ __launch_bounds__(256) void k_loss_join(const float* acc, int splits, int N, int K,
                                                   uint16_t* out, int64_t out_stride) {
  const int64_t total = (int64_t)N * K, stride = (int64_t)gridDim.x * 1024;
  for (int64_t i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x); i < total; i += stride) {
    lf32x4 s = *(const lf32x4*)(acc + i);
#pragma unroll 8
    for (int q = 1; q < splits; ++q) s += *(const lf32x4*)(acc + q * total + i);
    const float f[4] = {s[0], s[1], s[2], s[3]};
    const int64_t n = i / K;
    *(uint2*)(out + n * out_stride + (i - n * K)) = loss_pack4(f);
  }
}

// ---- host --------------------------------------------------------------------------------
constexpr int LG_CUS = 256;
// p of one vocabulary piece (256 of the vocabulary's rows are the least: more from 2^20 rows on)
constexpr int64_t LOSS_P_BYTES = (int64_t)512 << 20;

static inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static inline int64_t up256(int64_t b) { return (b + 255) & ~(int64_t)255; }

enum LossShape { LS_256x256, LS_256x128, LS_256x64, LS_128x128, LS_128x64 };
static int shape_m(LossShape s) { return s == LS_128x128 || s == LS_128x64 ? 128 : 256; }
static int shape_n(LossShape s) {
  return s == LS_256x256 ? 256 : s == LS_256x64 || s == LS_128x64 ? 64 : 128;
}
// rows of the M side that one wave has (its vocabulary slice in LM_STATS)
static int shape_slice(LossShape s) {
  return s == LS_256x256 ? 128 : s == LS_128x64 || s == LS_256x64 ? 32 : 64;
}
// about how long a step (64 along the reduction) of a CU's round of tiles takes, us, and how
// many tiles a round has
static double shape_us(LossShape s) {
  return s == LS_256x256 ? 1.7 : s == LS_256x128 ? 1.0 : s == LS_256x64 ? 0.7 : s == LS_128x128 ? 1.1 : 0.7;
}
static int64_t shape_round(LossShape s) { return shape_m(s) == 128 ? 2 * LG_CUS : LG_CUS; }

// us a step that an M x N result, `splits` times over, takes in tiles of one shape
static double shape_cost(LossShape s, int64_t m, int64_t n, int64_t splits) {
  const int64_t tiles = ceil_div(m, shape_m(s)) * ceil_div(n, shape_n(s)) * splits;
  // (a round of few 128-row tiles leaves each a CU of its own)
  const double alone = tiles <= LG_CUS && shape_m(s) == 128 ? 0.6 : 1.0;
  return alone * shape_us(s) * (double)ceil_div(tiles, shape_round(s));
}

// The shape whose rounds take least.
static LossShape loss_shape(int64_t m, int64_t n, int64_t splits, bool head) {
  LossShape best = LS_256x256;
  double least = 1e30;
  for (LossShape s : {LS_256x256, LS_256x128, LS_256x64, LS_128x128, LS_128x64}) {
    if (head && s != LS_256x256 && s != LS_128x128) continue;
    const double us = shape_cost(s, m, n, splits);
    if (us < least * 0.999) least = us, best = s;
  }
  return best;
}

// Of `v` vocabulary rows by `other` in large tiles, those (a multiple of 256) of whole rounds,
// where the rest takes half a round of large ones or less in smaller tiles (`rest`) and a launch of
// its own; else all. (N = 1,003, V = 100,003, K = 2,056, 28 tiles past six rounds: the loss 478 ->
// 442 us; with two thirds of a round, N = 700, V = 50,000, K = 2,048: the gradients 486 -> 497.)
static int64_t loss_main(LossShape shape, int64_t v, int64_t other, int64_t steps, bool head,
                         LossShape& rest) {
  if (shape != LS_256x256) return v;
  const int64_t row = ceil_div(other, 256), rounds = ceil_div(v, 256) * row / LG_CUS;
  const int64_t main = rounds * LG_CUS / row * 256;
  if (main == 0 || main >= v) return v;
  rest = head ? loss_shape(other, v - main, 1, true) : loss_shape(v - main, other, 1, false);
  const double all = shape_cost(shape, v, other, 1), large = shape_cost(shape, main, other, 1);
  const double small = head ? shape_cost(rest, other, v - main, 1) : shape_cost(rest, v - main, other, 1);
  return small <= 0.5 * shape_us(LS_256x256) && (all - large - small) * steps > 20.0 ? main : v;
}

struct LossPlan {
  LossShape prob;  // tile of the logits' products
  LossShape hid;   // of d_hidden's
  LossShape head;  // of d_lm_head's
  int piece;       // vocabulary rows a piece (a multiple of 256)
  int splits;      // d_hidden: parts of a piece's vocabulary
  int64_t part, tlogit, scale, p, acc, rows, bytes;  // offsets into the workspace
};

// slices that LM_STATS writes
static int64_t loss_slices(int64_t V, int64_t N, int64_t K, LossShape s) {
  auto slices = [](int64_t v, LossShape t) { return ceil_div(v, shape_m(t)) * (shape_m(t) / shape_slice(t)); };
  LossShape rest = s;
  const int64_t main = loss_main(s, V, N, ceil_div(K, LG_BK), false, rest);
  return slices(main, s) + (main < V ? slices(V - main, rest) : 0);
}

// p's rows end a line apart from a whole piece: rows a multiple of 8 KB apart, as pieces that
// make whole rounds have them, meet in few memory channels.
static int64_t loss_p_stride(int piece) { return piece + 64; }

static LossPlan loss_plan(int N, int K, int V, bool hid, bool head) {
  LossPlan q{};
  q.prob = loss_shape(V, N, 1, false);
  int64_t off = 0;
  auto take = [&](int64_t bytes) {
    const int64_t at = off;
    off += up256(bytes);
    return at;
  };
  if (!hid && !head) {
    q.part = take(loss_slices(V, N, K, q.prob) * N * (int64_t)sizeof(float2));
    q.tlogit = take(4 * (int64_t)N);
    q.bytes = off;
    return q;
  }
  // The piece whose rounds of 256 x 256 tiles take least over all pieces: equal ones, or ones
  // that end with whole rounds. (N = 4,096, V = 151,936, K = 5,120: 256 + 256 + 82 tiles of the
  // vocabulary take 38 rounds of logits' products, three pieces of 198 take 39.)
  const int64_t vt = ceil_div(V, 256), tn = ceil_div(N, 256), kt = ceil_div(K, 256);
  const int64_t most = LOSS_P_BYTES / (512 * (int64_t)N) > 1 ? LOSS_P_BYTES / (512 * (int64_t)N) : 1;
  int64_t best = -1, tiles = vt;
  auto offer = [&](int64_t t) {
    if (t < 1 || t > most) return;
    const int64_t full = ceil_div(vt, t) - 1, last = vt - t * full;
    auto rounds = [&](int64_t side) {
      return full * ceil_div(t * side, LG_CUS) + ceil_div(last * side, LG_CUS);
    };
    const int64_t cost = rounds(tn) * K + (head ? rounds(kt) * N : 0);
    if (best < 0 || cost < best) best = cost, tiles = t;
  };
  const int64_t np = ceil_div(vt, most);
  for (int64_t p = np; p < np + 3; ++p) offer(ceil_div(vt, p));
  int64_t whole = LG_CUS;  // tiles of the vocabulary that make whole rounds
  while (whole > 1 && whole / 2 * tn % LG_CUS == 0) whole /= 2;
  if (np > 1)
    for (int64_t t = most / whole * whole, e = t - 4 * whole; t > e; t -= whole) offer(t);
  q.piece = (int)(tiles * 256);
  q.prob = loss_shape(V < q.piece ? V : q.piece, N, 1, false);
  q.head = loss_shape(K, V < q.piece ? V : q.piece, 1, true);
  // d_hidden's reduction is split until its tiles fill the CUs; each split costs a pass over
  // its float32 sums
  const int64_t steps = ceil_div(q.piece, LG_BK);
  double least = 1e30;
  for (int s = 1; s <= 64 && s <= steps; ++s) {
    const LossShape shape = loss_shape(K, N, s, false);
    const double us = shape_cost(shape, K, N, s) * (double)ceil_div(steps, s) + 8.0 * s * N * (double)K / 4e6;
    if (us < least) least = us, q.splits = s, q.hid = shape;
  }
  q.scale = take(4);
  q.p = take((int64_t)N * loss_p_stride(q.piece) * 2);
  if (hid) q.acc = take((int64_t)q.splits * N * K * 4);
  if (head) q.rows = take((int64_t)N * K * 2);
  q.bytes = off;
  return q;
}

// Rows whose logits' product is one launch: a launch has fewer than 2^32 threads (one of more runs
// some of its workgroups only, without an error), and this many rows' tiles half of that. The
// gradients' products take more only beyond what memory holds.
static int loss_launch_rows(int V) { return (int)(((int64_t)1 << 22) / ceil_div(V, 256) * 256); }

int64_t loss_workspace(int N, int K, int V, bool hid, bool head) {
  const int64_t bytes = loss_plan(N, K, V, hid, head).bytes;
  const int most = loss_launch_rows(V);
  if (hid || head || N <= most) return bytes;
  const int64_t full = loss_plan(most, K, V, false, false).bytes;
  const int64_t last = loss_plan((N - 1) % most + 1, K, V, false, false).bytes;
  return full > last ? full : last;
}

template <int MODE, int WM, int WN, int TM, int TN, int R>
static void loss_gemm_as(LossGemm g, int64_t m, int64_t n, hipStream_t st) {
  g.tiles_m = (int)ceil_div(m, WM * TM * 16);
  g.tiles_n = (int)ceil_div(n, WN * TN * 16);
  const dim3 grid((unsigned)((int64_t)g.tiles_m * g.tiles_n * g.splits));
  hipLaunchKernelGGL((k_loss_gemm<MODE, WM, WN, TM, TN, R>), grid, dim3(WM * WN * WAVE), 0, st, g);
}

template <int MODE>
static void loss_gemm(const LossGemm& g, LossShape s, int64_t m, int64_t n, hipStream_t st) {
  if (s == LS_256x256) loss_gemm_as<MODE, 2, 4, 8, 4, 2>(g, m, n, st);
  else if (s == LS_128x128) loss_gemm_as<MODE, 2, 2, 4, 4, 2>(g, m, n, st);
  else if constexpr (MODE != LM_DHEAD) {
    if (s == LS_256x128) loss_gemm_as<MODE, 4, 2, 4, 4, 3>(g, m, n, st);
    else if (s == LS_256x64) loss_gemm_as<MODE, 8, 1, 2, 4, 3>(g, m, n, st);
    else loss_gemm_as<MODE, 4, 1, 2, 4, 3>(g, m, n, st);
  }
}

// The products along the vocabulary (M side; LM_DHEAD: N side): large tiles, then the rest of them.
template <int MODE>
static void loss_gemm_vocab(const LossGemm& g, LossShape s, int64_t v, int64_t other, hipStream_t st) {
  constexpr bool HEAD = MODE == LM_DHEAD;
  LossShape rest = s;
  const int64_t main = loss_main(s, v, other, ceil_div(g.red, LG_BK), HEAD, rest);
  loss_gemm<MODE>(g, s, HEAD ? other : main, HEAD ? main : other, st);
  if (main == v) return;
  LossGemm t = g;
  t.v0 += (int)main;
  if constexpr (HEAD) {
    t.b.p += main;
    t.b.rows -= (int)main;
    t.out16 += main * g.out_stride;
  } else {
    t.a.p += main * g.a.stride;
    t.a.rows -= (int)main;
    if constexpr (MODE == LM_STATS) t.part += main / shape_slice(s) * g.b.rows;
    else t.out16 += main;
  }
  loss_gemm<MODE>(t, rest, HEAD ? other : v - main, HEAD ? v - main : other, st);
}

static void loss_rows(const void* hidden, int64_t hs, int N, int K, const void* W, int64_t ws, int V,
                      const int32_t* targets, int ignore_index, void* workspace, float* loss,
                      float* lse, int32_t* status, hipStream_t st) {
  const LossPlan q = loss_plan(N, K, V, false, false);
  uint8_t* w8 = (uint8_t*)workspace;
  LossGemm g{};
  g.a = LossOperand{(const uint16_t*)W, ws, V};
  g.b = LossOperand{(const uint16_t*)hidden, hs, N};
  g.red = K;
  g.split_red = (int)(ceil_div(K, LG_BK) * LG_BK);
  g.splits = 1;
  g.V = V;
  g.ignore_index = ignore_index;
  g.targets = targets;
  g.part = (float2*)(w8 + q.part);
  g.tlogit = (float*)(w8 + q.tlogit);
  loss_gemm_vocab<LM_STATS>(g, q.prob, V, N, st);
  const int slices = (int)loss_slices(V, N, K, q.prob);
  // (512 rows of 1,187 slices: two tokens a workgroup 8.2 us, eight 5.5; 200 rows of 782: 4.1 and
  // 4.5; 4,096 rows: eight 13.8, sixteen 9.2)
  auto rows = [&](auto kernel, int tokens) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(N, tokens)), dim3(256), 0, st, g.part, slices, N,
                       g.tlogit, targets, ignore_index, V, loss, lse, status);
  };
  if (N >= 1024) rows(k_loss_rows<16>, 16);
  else if (N >= 256) rows(k_loss_rows<8>, 8);
  else rows(k_loss_rows<2>, 2);
}

hipError_t launch_loss(const void* hidden, int64_t hs, int N, int K, const void* W, int64_t ws, int V,
                       const int32_t* targets, int ignore_index, void* workspace, float* loss,
                       float* lse, int32_t* status, hipStream_t st) {
  const int most = loss_launch_rows(V);
  for (int n = 0; n < N; n += most)
    loss_rows((const uint16_t*)hidden + n * hs, hs, min(most, N - n), K, W, ws, V, targets + n,
              ignore_index, workspace, loss + n, lse ? lse + n : nullptr, status ? status + n : nullptr, st);
  return hipGetLastError();
}

hipError_t launch_loss_grad(const void* hidden, int64_t hs, int N, int K, const void* W, int64_t ws,
                            int V, const int32_t* targets, int ignore_index, const float* lse,
                            const float* grad_loss, const float* grad_lse, void* workspace,
                            void* d_hidden, int64_t dhs, void* d_head, int64_t dws,
                            hipStream_t st) {
  if (N == 0) {  // no reduction: the projection's gradient is zero
    LossGemm z{};
    z.a.rows = K;
    z.b.rows = V;
    z.splits = 1;
    z.out16 = (uint16_t*)d_head;
    z.out_stride = dws;
    if (d_head) loss_gemm<LM_DHEAD>(z, LS_256x256, K, V, st);
    return hipGetLastError();
  }
  const LossPlan q = loss_plan(N, K, V, d_hidden != nullptr, d_head != nullptr);
  uint8_t* w8 = (uint8_t*)workspace;
  uint16_t *p = (uint16_t*)(w8 + q.p), *rows = (uint16_t*)(w8 + q.rows);
  if (d_head)
    hipLaunchKernelGGL(k_loss_rows_in, dim3((unsigned)N), dim3(256), 0, st, (const uint16_t*)hidden,
                       hs, N, K, targets, ignore_index, V, rows);
  for (int v0 = 0; v0 < V; v0 += q.piece) {
    const int vn = min(q.piece, V - v0);
    const uint16_t* wv = (const uint16_t*)W + (int64_t)v0 * ws;
    LossGemm g{};
    g.a = LossOperand{wv, ws, vn};
    g.b = LossOperand{(const uint16_t*)hidden, hs, N};
    g.red = K;
    g.split_red = (int)(ceil_div(K, LG_BK) * LG_BK);
    g.splits = 1;
    g.v0 = v0;
    g.V = V;
    g.ignore_index = ignore_index;
    g.targets = targets;
    g.lse = lse;
    g.grad_loss = grad_loss;
    g.grad_lse = grad_lse;
    g.scale = (float*)(w8 + q.scale);
    g.out16 = p;
    g.out_stride = loss_p_stride(q.piece);
    loss_gemm_vocab<LM_PROB>(g, q.prob, vn, N, st);
    if (d_hidden) {
      LossGemm h{};
      h.a = LossOperand{wv, ws, K};
      h.b = LossOperand{p, loss_p_stride(q.piece), N};
      h.red = vn;
      h.splits = q.splits;
      h.split_red = (int)(ceil_div(ceil_div(vn, LG_BK), q.splits) * LG_BK);
      h.scale = g.scale;
      h.out32 = (float*)(w8 + q.acc);
      h.out_stride = K;
      h.accumulate = v0 > 0;
      loss_gemm<LM_DHID>(h, q.hid, K, N, st);
    }
    if (d_head) {
      LossGemm h{};
      h.a = LossOperand{rows, K, K};
      h.b = LossOperand{p, loss_p_stride(q.piece), vn};
      h.red = N;
      h.splits = 1;
      h.split_red = (int)(ceil_div(N, LG_BK) * LG_BK);
      h.scale = g.scale;
      h.out16 = (uint16_t*)d_head + (int64_t)v0 * dws;
      h.out_stride = dws;
      loss_gemm_vocab<LM_DHEAD>(h, q.head, vn, K, st);
    }
  }
  if (d_hidden) {
    const int64_t blocks = min(ceil_div((int64_t)N * K, 1024), (int64_t)1 << 22);
    hipLaunchKernelGGL(k_loss_join, dim3((unsigned)blocks), dim3(256), 0, st,
                       (const float*)(w8 + q.acc), q.splits, N, K, (uint16_t*)d_hidden, dhs);
  }
  return hipGetLastError();
}

}  // namespace strim
