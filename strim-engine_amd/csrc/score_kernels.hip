// score_kernels.hip — what a row of logits says about its tokens, and the gradient that goes back into it.
//
//   z[v] = x[v] / T on allowed ids, -inf elsewhere;  lse = log sum_v exp(z[v])
//   logprob[t] = z[t] - lse,  H = -sum_v p log p with p = exp(z - lse),  the first `top` ids in token order
//   dx[v] = 1/T (sum_s g[s] ([v = t_s] - p[v]) - gH p[v] (log p[v] + H) + gL p[v])
//
// k_scores reads the logits once: per lane the running maximum m, s = sum 2^y and u = sum y 2^y with y =
// (x - m) log2(e) / T, from which lse = m / T + log s and H = log s - log(2) u / s, and the row's
// alternatives (top.hpp). A row is one workgroup's where there are many, else in parts that
// k_scores_join merges. Bound by the reading where rows are many (V = 151,936, bf16, R = 2,048: 105 us, 5.9 TB/s, with
// 64 alternatives 124; float32, R = 1,003, V = 100,003: 76 us, 5.3), by two launches' round trips where they are few
// (one row with 20 alternatives 11.3 us, 64 rows with five 16.9). The join is a launch of its own: a last part that
// waited for the others' results would need a device-scope release, which costs more.
#include <type_traits>

#include "kernels.hpp"
#include "rows.hpp"
#include "score.hpp"
#include "top.hpp"

namespace strim {

namespace {

constexpr int SC_T = TOP_T;                    // threads of a workgroup
constexpr int SC_U = TOP_STEP * 2 / (8 * SC_T);  // vectors of eight tokens a lane has of a tile
constexpr int SC_TILE = 8 * SC_U * SC_T;       // tokens a tile

// What a part of a row leaves for the join: its statistics and ScoreParts::room entries of its alternatives
// (TOP_NONE past the last).
struct ScoreParts {
  int32_t parts, tiles;  // parts of a row; tiles of a part
  int32_t room;
  RowStat* part;         // [R][parts]
  uint64_t* keys;        // [R][parts][room]
};

__device__ __forceinline__ bool allowed_at(const uint32_t* mask, int v) {
  return !mask || ((mask[v >> 5] >> (v & 31)) & 1u);
}

// A given token and its logit, -inf where the mask forbids it; the thread's own (S <= SC_T). Asked for before
// the row's statistics are known.
struct Given {
  float x;
  bool given, inside;
};
template <int DT>
__device__ __forceinline__ Given given_of(const ScoreArgs& a, int64_t r) {
  const char* row = (const char*)a.logits + r * a.stride * RowVec<DT>::SIZE;
  const uint32_t* mask = a.mask ? a.mask + r * a.mask_stride : nullptr;
  Given o{-INFINITY, false, false};
  if ((int)threadIdx.x < a.S) {
    const int t = a.tokens[r * a.S + threadIdx.x];
    o.given = t != a.ignore_index;
    o.inside = t >= 0 && t < a.V;
    if (o.given && o.inside && allowed_at(mask, t)) o.x = token_at<DT>(row, t);
  }
  return o;
}

// The row's results from its statistics and the list that holds its first `top` keys.
__device__ __forceinline__ void score_finish(const ScoreArgs& a, int64_t r, RowStat st, Given t, TopList* l, int n) {
  const float nan = __builtin_nanf("");
  const bool bad = !(st.s < INFINITY), empty = !bad && st.s == 0.0f;
  const float ls = logf(st.s);
  // (not from lse, which is rounded to the largest logit's spacing)
  auto logprob = [&](float x) { return (x - st.m) / a.T - ls; };
  if ((int)threadIdx.x < a.S)
    a.logprobs[r * a.S + threadIdx.x] = !(t.given && t.inside) ? 0.0f : bad ? nan : empty ? -INFINITY : logprob(t.x);
  const bool unknown = a.status && __syncthreads_or(t.given && !t.inside);
  if (threadIdx.x == 0) {
    a.entropy[r] = bad ? nan : empty ? 0.0f : ls - 0.69314718055994531f * (st.u / st.s);
    a.lse[r] = bad ? nan : empty ? -INFINITY : st.m / a.T + ls;
    if (a.status)
      a.status[r] = bad ? STRIM_ENONFINITE : empty ? STRIM_EEMPTY : unknown ? STRIM_EINVAL : STRIM_OK;
  }
  if (!l) return;
  int32_t* ids = a.top_ids + r * a.top;
  float* lps = a.top_logprobs + r * a.top;
  if (bad) n = 0;
  for (int k = n + (int)threadIdx.x; k < a.top; k += SC_T) {
    ids[k] = -1;
    lps[k] = bad ? nan : -INFINITY;
  }
  top_order(*l, n, a.top, [&](int k, uint64_t key) {
    ids[k] = (int32_t)(uint32_t)key;
    lps[k] = logprob(fkey_desc_inv((uint32_t)(key >> 32)));
  });
}

// The workgroup's statistics in every thread.
__device__ __forceinline__ RowStat stat_block(RowStat st, float c, RowStat* scratch) {
  stat_wave(st, c);
  if ((threadIdx.x & (WAVE - 1)) == 0) scratch[threadIdx.x / WAVE] = st;
  __syncthreads();
  st = scratch[0];
#pragma unroll
  for (int i = 1; i < SC_T / WAVE; ++i) stat_merge(st, scratch[i], c);
  return st;
}

template <int DT, bool MASK, bool TOP>
__global__ __launch_bounds__(SC_T, DT == STRIM_DTYPE_BF16 ? 8 : 6) void k_scores(const ScoreArgs a, const ScoreParts q) {
  __shared__ RowStat s_stat[SC_T / WAVE];
  __shared__ std::conditional_t<TOP, TopList, char> s_list;
  TopList* const s_top = (TopList*)&s_list;  // (unused without TOP)
  const int64_t r = blockIdx.x / q.parts;
  const int p = blockIdx.x - (int)r * q.parts, lane = threadIdx.x & (WAVE - 1), wave = wave_id();
  const char* row = (const char*)a.logits + r * a.stride * RowVec<DT>::SIZE;
  const uint32_t* mask = MASK ? a.mask + r * a.mask_stride : nullptr;
  const float c = LOG2E / a.T;
  const int t0 = p * q.tiles * SC_TILE, t1 = min(a.V, t0 + q.tiles * SC_TILE);
  RowVec<DT> next[SC_U];
  uint32_t ok[SC_U];
  auto request = [&](int t) {
#pragma unroll
    for (int u = 0; u < SC_U; ++u) {
      const int v0 = t + 8 * WAVE * (u * (SC_T / WAVE) + wave);
      if (t + SC_TILE <= a.V) next[u].template load<true>(row, v0, lane);
      else next[u].load_to(row, v0, lane, a.V);
      if (MASK) ok[u] = allowed8<DT>(mask, v0, lane, a.V);
    }
  };
  request(t0);
  TopRun top;
  if constexpr (TOP) top.init(s_top[0], a.top);
  RowStat st{-INFINITY, 0.0f, 0.0f};
  for (int t = t0; t < t1;) {
    bool fits = true;
    for (; fits && t < t1; t += SC_TILE) {
      float x[8 * SC_U], mv[SC_U], mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < SC_U; ++u) {
        mv[u] = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float f = next[u].at(j);
          if (MASK) f = (ok[u] >> j) & 1u ? f : -INFINITY;
          x[8 * u + j] = f;
          mv[u] = fmaxf(mv[u], f);
        }
        mx = fmaxf(mx, mv[u]);
      }
      if (t + SC_TILE < t1) request(t + SC_TILE);
      stat_add<8 * SC_U, true>(st, x, mx, c);
      if constexpr (TOP)
        fits = top.add<SC_U>(s_top[0], x, mv, st.m, t + 8 * WAVE * wave + RowVec<DT>::first(lane), RowVec<DT>::step);
    }
    if constexpr (TOP)
      if (!fits) {  // the last tile again, slot by slot (out of the loop, for its registers' sake)
        const int s = t - SC_TILE;
        auto load = [&](int u, float (&x)[8]) {
          const int v0 = s + 8 * WAVE * (u * (SC_T / WAVE) + wave);
          RowVec<DT> q;
          q.load_to(row, v0, lane, a.V);
          const uint32_t in = MASK ? allowed8<DT>(mask, v0, lane, a.V) : 0xFFu;
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = (in >> j) & 1u ? q.at(j) : -INFINITY;
        };
        top_slots<SC_U>(top, s + 8 * WAVE * wave + RowVec<DT>::first(lane), load, RowVec<DT>::step);
      }
  }
  const float most = st.m;
  Given given{};
  if (q.parts == 1) given = given_of<DT>(a, r);
  if constexpr (TOP) top.leave(s_top[0]);
  st = stat_block(st, c, s_stat);
  if (q.parts == 1) {
    int n = 0;
    if constexpr (TOP) n = top.gather(s_top[0], most);
    stat_exact(st, c);
    return score_finish(a, r, st, given, TOP ? s_top : nullptr, n);
  }
  if (threadIdx.x == 0) q.part[r * q.parts + p] = st;
  if constexpr (TOP) {
    // (short lists go to the join as they are: R = 64, V = 151,936, M = 5 16.9 us, with every list cut 20.3)
    uint64_t* out = q.keys + (r * q.parts + p) * q.room;
    int n;
    const int at = top.place(s_top[0], n);
    if (n <= q.room) {
      for (int i = lane; i < top.held; i += WAVE) out[at + i] = top.e[i];
    } else {
      n = top.gather(s_top[0], most);
      if (n <= q.room) {
        for (int i = threadIdx.x; i < n; i += SC_T) out[i] = s_top[0].e[i];
      } else {
        top_order(s_top[0], n, q.room, [&](int k, uint64_t key) {
          out[k] = top_entry(fkey_desc_inv((uint32_t)(key >> 32)), (int32_t)(uint32_t)key);
        });
        n = q.room;
      }
    }
    for (int i = n + (int)threadIdx.x; i < q.room; i += SC_T) out[i] = TOP_NONE;
  }
}

template <int DT, bool TOP>
__global__ __launch_bounds__(SC_T) void k_scores_join(const ScoreArgs a, const ScoreParts q) {
  __shared__ RowStat s_stat[SC_T / WAVE];
  __shared__ std::conditional_t<TOP, TopList, char> s_list;
  TopList* const s_top = (TopList*)&s_list;  // (unused without TOP)
  constexpr int Q = TOP_STEP / SC_T;         // entries a thread takes at a time
  const int64_t r = blockIdx.x;
  const float c = LOG2E / a.T;
  RowStat st{-INFINITY, 0.0f, 0.0f};
  if ((int)threadIdx.x < q.parts) st = q.part[r * q.parts + threadIdx.x];
  const uint64_t* keys = q.keys + r * q.parts * q.room;
  const int all = TOP ? q.parts * q.room : 0;
  uint64_t k[Q];
  auto request = [&](int i0) {
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const int at = i0 + i * SC_T + (int)threadIdx.x;
      k[i] = at < all ? keys[at] : TOP_NONE;
    }
  };
  if constexpr (TOP) request(0);
  const Given given = given_of<DT>(a, r);
  st = stat_block(st, c, s_stat);
  int n = 0;
  if constexpr (TOP) {
    uint32_t best = ~0u;
    for (int i0 = 0; i0 < all; i0 += TOP_STEP) {
      if (i0 > 0) request(i0);
#pragma unroll
      for (int i = 0; i < Q; ++i) best = min(best, fkey_desc(__uint_as_float((uint32_t)(k[i] >> 32))));
    }
    const uint32_t t = top_threshold(s_top[0], best, TOP_ALL, a.top, 0);
    const float floor = fkey_desc_inv(t);
    if (threadIdx.x == 0) s_top[0].n = 0;
    __syncthreads();
    for (int i0 = 0; i0 < all; i0 += TOP_STEP) {
      if (all > TOP_STEP) request(i0);
      if (n > TOP_T) {  // (lists full of ties)
        uint32_t unused = 0;
        n = top_reduce(s_top[0], n, a.top, unused);
        if (threadIdx.x == 0) s_top[0].n = n;
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < Q; ++i)
        if (__uint_as_float((uint32_t)(k[i] >> 32)) >= floor) s_top[0].e[atomicAdd(&s_top[0].n, 1)] = k[i];
      __syncthreads();
      n = __builtin_amdgcn_readfirstlane(s_top[0].n);
      __syncthreads();
    }
  }
  stat_exact(st, c);
  score_finish(a, r, st, given, TOP ? s_top : nullptr, n);
}

// The gradient: G = sum of the tokens' gradients, then d = p (gL - G - gH (log p + H)) / T everywhere and
// g / T more at the tokens. A wave finds its 512 tokens' given ones by one ballot of the list, which its
// lanes hold (two entries each), and hands each to the lane and element that it belongs to. One read and one
// write, both past the caches where the result is large: R = 1,003, V = 100,003, float32 150 us, 5.3 TB/s.
constexpr int SG_TILES = 4;  // tiles of eight tokens a thread that a workgroup takes

template <int DT, bool MASK, bool ENT>
__global__ __launch_bounds__(SC_T) void k_scores_grad(const ScoreGradArgs a, int parts) {
  const int64_t r = blockIdx.x / parts;
  const int p = blockIdx.x - (int)r * parts, lane = threadIdx.x & (WAVE - 1);
  const char* row = (const char*)a.logits + r * a.stride * RowVec<DT>::SIZE;
  char* out = (char*)a.d_logits + r * a.d_stride * RowVec<DT>::SIZE;
  const uint32_t* mask = MASK ? a.mask + r * a.mask_stride : nullptr;
  const int t0 = p * SG_TILES * 8 * SC_T, wave = wave_id();
  RowVec<DT> x[SG_TILES];
  uint32_t ok[SG_TILES];
#pragma unroll
  for (int u = 0; u < SG_TILES; ++u) {
    const int w0 = t0 + 8 * WAVE * (u * (SC_T / WAVE) + wave);
    x[u].template load_to<false, true>(row, w0, lane, a.V);
    if (MASK) ok[u] = allowed8<DT>(mask, w0, lane, a.V);
  }
  const float lse = a.lse[r], c = LOG2E / a.T, inv = 1.0f / a.T;
  const float gh = ENT ? a.grad_entropy[r] : 0.0f, H = ENT ? a.entropy[r] : 0.0f;
  int id[2];
  float g[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = lane + i * WAVE;
    id[i] = s < a.S ? a.tokens[r * a.S + s] : -1;
    if (id[i] == a.ignore_index || id[i] >= a.V) id[i] = -1;
    g[i] = id[i] >= 0 ? a.grad_logprobs[r * a.S + s] * inv : 0.0f;
  }
  const float G = wave_sum_f(g[0] + g[1]), top = (a.grad_lse ? a.grad_lse[r] * inv : 0.0f) - G;
  const bool empty = lse == -INFINITY;
  const float ref = lse * a.T;
#pragma unroll
  for (int u = 0; u < SG_TILES; ++u) {
    const int w0 = t0 + 8 * WAVE * (u * (SC_T / WAVE) + wave);
    if (w0 >= a.V) break;
    float d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y = x[u].at(j) - ref, p = hw_exp2(y * c);
      d[j] = ENT ? p * (top - gh * inv * (fmaxf(y * inv, -200.0f) + H)) : p * top;
    }
    // the given tokens among these 512, in the list's order
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint64_t hit = __ballot(id[i] >= 0 && (uint32_t)(id[i] - w0) < 8u * WAVE);
      while (hit) {
        const int l = __builtin_ctzll(hit);
        hit &= hit - 1;
        const int off = rl_i(id[i], l) - w0;
        const float more = rl_f(g[i], l);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          d[j] += lane == RowVec<DT>::lane_of(off) && j == RowVec<DT>::element_of(off) ? more : 0.0f;
      }
    }
    if (MASK)
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = (ok[u] >> j) & 1u ? d[j] : 0.0f;
    RowVec<DT> y;
    y.set(d);
    if (empty)
#pragma unroll
      for (int i = 0; i < RowVec<DT>::WORDS; ++i) y.w[i] = 0;
    y.store_to(out, w0, lane, a.V, a.stream);
  }
}

int64_t up16(int64_t b) { return (b + 15) & ~(int64_t)15; }
int64_t ceil_of(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Parts of a row: as many workgroups in all as the chip holds at once (eight a CU), one a row where there
// are that many rows.
ScoreParts score_parts(int R, int V, int top) {
  ScoreParts q{};
  const int64_t tiles = ceil_of(V, SC_TILE), each = ceil_of((int64_t)R * tiles, 2048);
  q.tiles = (int32_t)(each > tiles ? tiles : each);
  q.parts = (int32_t)ceil_of(tiles, q.tiles);
  q.room = top == 0 ? 0 : 2 * top > 32 ? 2 * top : 32;
  return q;
}

}  // namespace

int64_t scores_workspace(int R, int V, int top) {
  const ScoreParts q = score_parts(R, V, top);
  if (q.parts == 1) return 0;
  return up16((int64_t)R * q.parts * (int64_t)sizeof(RowStat)) + (int64_t)R * q.parts * q.room * 8;
}

hipError_t launch_scores(const ScoreArgs& a, bool bf16, void* workspace, hipStream_t st) {
  ScoreParts q = score_parts(a.R, a.V, a.top);
  if (q.parts > 1) {
    q.part = (RowStat*)workspace;
    q.keys = (uint64_t*)((char*)workspace + up16((int64_t)a.R * q.parts * (int64_t)sizeof(RowStat)));
  }
  const dim3 grid((unsigned)((int64_t)a.R * q.parts)), threads(SC_T);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, threads, 0, st, a, q); };
  auto join = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)a.R), threads, 0, st, a, q); };
  auto all = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (a.mask) a.top ? go(k_scores<DT, true, true>) : go(k_scores<DT, true, false>);
    else a.top ? go(k_scores<DT, false, true>) : go(k_scores<DT, false, false>);
    if (q.parts > 1) a.top ? join(k_scores_join<DT, true>) : join(k_scores_join<DT, false>);
  };
  if (bf16) all(std::integral_constant<int, STRIM_DTYPE_BF16>{});
  else all(std::integral_constant<int, STRIM_DTYPE_F32>{});
  return hipGetLastError();
}

hipError_t launch_scores_grad(const ScoreGradArgs& a, bool bf16, hipStream_t st) {
  const int parts = (int)ceil_of(a.V, 8 * SC_T * SG_TILES);
  // (a launch has fewer than 2^32 threads)
  const int most = (int)(((int64_t)1 << 23) / parts);
  for (int r0 = 0; r0 < a.R; r0 += most) {
    ScoreGradArgs b = a;
    b.stream = (int64_t)a.R * a.V * (bf16 ? 2 : 4) > ROWS_CACHED;
    const int64_t at = r0;
    b.R = a.R - r0 < most ? a.R - r0 : most;
    b.logits = (const char*)a.logits + at * a.stride * (bf16 ? 2 : 4);
    b.d_logits = (char*)a.d_logits + at * a.d_stride * (bf16 ? 2 : 4);
    if (a.mask) b.mask = a.mask + at * a.mask_stride;
    if (a.tokens) b.tokens = a.tokens + at * a.S;
    b.lse = a.lse + at;
    if (a.entropy) b.entropy = a.entropy + at;
    if (a.grad_logprobs) b.grad_logprobs = a.grad_logprobs + at * a.S;
    if (a.grad_entropy) b.grad_entropy = a.grad_entropy + at;
    if (a.grad_lse) b.grad_lse = a.grad_lse + at;
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)((int64_t)b.R * parts)), dim3(SC_T), 0, st, b, parts);
    };
    auto all = [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      if (a.mask) a.grad_entropy ? go(k_scores_grad<DT, true, true>) : go(k_scores_grad<DT, true, false>);
      else a.grad_entropy ? go(k_scores_grad<DT, false, true>) : go(k_scores_grad<DT, false, false>);
    };
    if (bf16) all(std::integral_constant<int, STRIM_DTYPE_BF16>{});
    else all(std::integral_constant<int, STRIM_DTYPE_F32>{});
  }
  return hipGetLastError();
}

}  // namespace strim
