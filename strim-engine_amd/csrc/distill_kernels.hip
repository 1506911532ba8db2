// distill_kernels.hip — distillation from a teacher's top logits: a student's rows x [V] against the
// alternatives (id_m, log-probability t_m), m < M.
//
//   p_m = softmax of t_m over the alternatives, r = 0; or (tail) p_m = exp(t_m), r = max(0, 1 - sum p)
//   q = softmax(x / T);  loss = sum_m p_m (log p_m - log q[id_m]) + r (log r - log q_rest)
//   dx[v] = w / T (q[v] (P + r - [v no alternative] r / q_rest) - sum of p_m with id_m = v),  P = sum p
//
// What needs the whole row is one softmax statistic: of all its tokens, or (tail) of those that are no
// alternative, so that q_rest is no difference of near numbers; the alternatives' own logits are looked
// up. Those M numbers are in 64 bits: a small loss is the difference of much larger terms.
//
// k_distill_step has a row in one workgroup between the statistic and the gradient: what registers and LDS hold
// of it is read once (all of 32,768 tokens; of 151,936 three quarters in bf16), the rest twice, all written once.
// Bound by HBM (V = 151,936, N = 4,096, bf16: 547 us for the 2.5 GB of one read and one write, 4.6 TB/s, a copy's
// 527; N = 96, V = 32,768: 10.3 us, a load, a store and the alternatives' chain of about 3 us between). Few rows over
// a long vocabulary, a loss or a gradient alone: k_distill_stat over parts of the rows (N = 500, V = 50,021, float32:
// 18.6 us, 5.4 TB/s), k_distill_join, k_distill_grad; a step so reads the logits twice (N = 64, V = 151,936, bf16: 8.9
// + 8.1 + 7.4 us; the gradient alone 14.6).
#include <type_traits>

#include "kernels.hpp"
#include "rows.hpp"
#include "score.hpp"

namespace strim {

namespace {

constexpr int DI_T = 256;                 // threads of the parts' workgroups
constexpr int DI_U = 4;                   // vectors of eight tokens a thread has of a tile
constexpr int DI_TILE = 8 * DI_U * DI_T;  // tokens a tile
constexpr int DI_M = STRIM_SCORE_MAX_LIST;

// A row's alternatives as a wave holds them: entry lane + 64 i in each lane, id -1 where there is none.
struct Alternatives {
  int id[2];
  float lp[2];
  bool known;  // no id past the vocabulary
  bool any;    // (and an alternative)
};
__device__ __forceinline__ Alternatives alternatives_of(const DistillArgs& a, int64_t r) {
  const int lane = threadIdx.x & (WAVE - 1);
  Alternatives o;
  bool past = false, any = false;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int m = lane + i * WAVE;
    o.id[i] = m < a.M ? a.ids[r * a.M + m] : -1;
    o.lp[i] = m < a.M ? a.logprobs[r * a.M + m] : -INFINITY;
    past |= o.id[i] >= a.V;
    if (o.lp[i] == -INFINITY) o.id[i] = -1;
    any |= o.id[i] >= 0;
  }
  o.known = __ballot(past) == 0;
  o.any = o.known && __ballot(any) != 0;
  return o;
}

// Each entry that is among the wave's 512 tokens from w0 on, in the list's order: f(lane, element, entry's
// lane, i).
template <int DT, class F>
__device__ __forceinline__ void each_hit(const int (&id)[2], int w0, F f) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint64_t hit = __ballot((uint32_t)(id[i] - w0) < 8u * WAVE);  // (an id of -1 is never)
    while (hit) {
      const int l = __builtin_ctzll(hit);
      hit &= hit - 1;
      const int off = rl_i(id[i], l) - w0;
      f(RowVec<DT>::lane_of(off), RowVec<DT>::element_of(off), l, i);
    }
  }
}
template <int DT>
__device__ __forceinline__ void without_hits(float (&x)[8], const int (&id)[2], int w0) {
  const int lane = threadIdx.x & (WAVE - 1);
  each_hit<DT>(id, w0, [&](int at, int e, int, int) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (lane == at && j == e) x[j] = -INFINITY;
  });
}

// A row's teacher: the entries' probabilities (0 where there is none), log p_m = lp_m - shift, P and r. The
// exponentials are float32 ones, the sums and differences double: an error that the p_m share with r moves
// a small loss by its product with the loss's own size.
struct Teacher {
  float p[2];
  double shift, mass, r;
};
__device__ __forceinline__ Teacher teacher_of(const Alternatives& o, bool tail) {
  Teacher t;
  float mx = 0.0f;
  if (!tail)
    mx = wave_max_f(fmaxf(o.id[0] >= 0 ? o.lp[0] : -INFINITY, o.id[1] >= 0 ? o.lp[1] : -INFINITY));
#pragma unroll
  for (int i = 0; i < 2; ++i) t.p[i] = o.id[i] >= 0 ? expf(o.lp[i] - mx) : 0.0f;
  const double sum = wave_sum((double)t.p[0] + (double)t.p[1]);
  t.mass = tail ? sum : 1.0;
  t.r = tail ? fmax(0.0, 1.0 - sum) : 0.0;
  t.shift = 0.0;
  if (!tail) {
    t.shift = mx + log(sum);
#pragma unroll
    for (int i = 0; i < 2; ++i) t.p[i] = (float)(t.p[i] / sum);
  }
  return t;
}

// Which entries are the first with their id, and those entries' p with the later ones' added. One wave.
__device__ __forceinline__ void merge_repeats(const Alternatives& o, int M, bool (&first)[2], float (&p)[2]) {
  const int lane = threadIdx.x & (WAVE - 1);
  float sum[2] = {0.0f, 0.0f};
  first[0] = o.id[0] >= 0;
  first[1] = o.id[1] >= 0;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    for (int l = 0; l < min(WAVE, M - h * WAVE); ++l) {
      const int id = rl_i(o.id[h], l);
      const float more = rl_f(p[h], l);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (id == o.id[i]) {
          sum[i] += more;
          if (h < i || (h == i && l < lane)) first[i] = false;
        }
    }
#pragma unroll
  for (int i = 0; i < 2; ++i) p[i] = sum[i];
}

// The teacher's remaining mass: where nothing lies outside the ids, one that float32 log-probabilities do not
// tell from none is none.
__device__ __forceinline__ double bucket_of(double r, bool empty) { return empty && r < 0x1p-20 ? 0.0 : r; }

// A row's numbers from the statistic: the loss; `ls` = log sum exp((x - top) / T) and log q_rest; for the tokens'
// gradients the same against their own largest logit `ref` (with a tail the rest's): `ls_ref` of all, `ls_rest` of
// the rest. x: the entries' logits. By one wave, every lane the same.
struct RowNumbers {
  double loss, top, ls, log_rest, ref, ls_ref, ls_rest;
};
__device__ __forceinline__ RowNumbers numbers_of(const Alternatives& o, const Teacher& t, const bool (&first)[2],
                                                 const float (&x)[2], RowStat st, float T, bool tail) {
  const int lane = threadIdx.x & (WAVE - 1);
  RowNumbers n;
  n.top = st.m;
  double all = st.s, far = 0.0;
  if (tail) {
    n.top = wave_max_f(fmaxf(st.m, fmaxf(first[0] ? x[0] : -INFINITY, first[1] ? x[1] : -INFINITY)));
    const float ref = stat_ref((float)n.top);
    double in = 0.0;
#pragma unroll
    for (int i = 0; i < 2; ++i) in += first[i] ? (double)expf((x[i] - ref) / T) : 0.0;
    in = wave_sum(in);
    far = ((double)st.m - ref) / T;
    all = (st.m == -INFINITY ? (double)st.s : (double)st.s * exp(far)) + in;
  }
  // the three logarithms by three lanes
  const double l = log(lane == 0 ? all : lane == 1 ? (double)st.s : t.r);
  n.ls = rl_d(l, 0);
  // (a rest whose share vanishes in 64 bits keeps its logarithm)
  n.log_rest = !tail ? 0.0 : st.m == -INFINITY ? -(double)INFINITY : far + rl_d(l, 1) - n.ls;
  n.ref = tail ? (double)stat_ref(st.m) : n.top;
  n.ls_ref = tail && st.m == -INFINITY ? 0.0 : n.ls - far;  // (no rest: no token that takes it)
  n.ls_rest = rl_d(l, 1);
  double loss = 0.0;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (o.id[i] >= 0 && !(t.p[i] == 0.0f))
      loss += t.p[i] * (((double)o.lp[i] - t.shift) - (((double)x[i] - n.top) / T - n.ls));
  n.loss = wave_sum(loss);
  if (bucket_of(t.r, st.m == -INFINITY) > 0.0) n.loss += t.r * (rl_d(l, 2) - n.log_rest);
  return n;
}

// What the gradient takes of a row: sign 2^y with y = (x - ref) c + k at every token, but at the alternatives
// in 2^y' - p, y' = (x - top) c + kq. (k and kq are rounded to float32 and have to be small: each goes with the largest
// logit of its own tokens.) bf16 results are taken as 2^(x c + b), b = k - ref c, where |b| is below 2^11 (`near`): b's
// rounding is then at most 2^-14 of an exponent, 2^-14.5 of a result, theirs 2^-9. It grows with b, and so with the
// largest logit over T.
struct GradRow {
  float top, ref, k, kq, in, b;
  uint32_t sign;  // 0 or 0x80008000
  int16_t near;
  int16_t dead;   // the row has no gradient
};
// w = weight / T
__device__ __forceinline__ GradRow grad_row(bool any, const Teacher& t, const RowNumbers& n, double w, float c) {
  constexpr double L2E = 1.4426950408889634074;
  GradRow g;
  g.dead = !any || w == 0.0;
  const double in = w * (t.mass + bucket_of(t.r, n.log_rest == -INFINITY));
  double all = in, ls = n.ls_ref;
  if (t.r > 0.0 && n.log_rest > -INFINITY) {  // (nothing lies outside where q_rest is 0)
    if (n.log_rest > -600.0) {
      all = in - w * t.r * exp(-n.log_rest);
    } else {
      all = -w * t.r;
      ls = n.ls_rest;
    }
  }
  const double k = log2(fabs(all)) - ls * L2E;
  g.top = (float)n.top;
  g.ref = (float)n.ref;
  g.kq = (float)(-n.ls * L2E);
  g.k = (float)k;
  g.in = (float)in;
  g.b = (float)(k - n.ref * c);
  g.near = fabsf(g.b) < 0x1p11f;  // (not where it is a NaN)
  g.sign = all < 0.0 ? 0x80008000u : 0u;
  return g;
}
// The numbers that the gradient takes from lse and log q_rest as float32 holds them.
__device__ __forceinline__ RowNumbers numbers_from(double lse, double log_rest, bool tail, float T) {
  constexpr double MOST = 3.40282346638528859812e38;
  auto near_to = [&](double z) { return (double)(float)fmax(-MOST, fmin(MOST, z * T)); };
  RowNumbers n{};
  n.log_rest = tail ? log_rest : 0.0;
  const double rest = log_rest > -INFINITY ? lse + log_rest : lse;
  n.top = near_to(lse);
  n.ls = lse - n.top / T;
  n.ref = tail ? near_to(rest) : n.top;
  n.ls_ref = lse - n.ref / T;
  n.ls_rest = rest - n.ref / T;
  return n;
}

// Eight tokens' gradients, as of no alternatives.
template <int DT>
__device__ __forceinline__ RowVec<DT> grad_of(const RowVec<DT>& x, const GradRow& g, float c) {
  float d[8];
  if (DT == STRIM_DTYPE_BF16 && g.near) {
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = hw_exp2(fma_f(x.at(j), c, g.b));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = hw_exp2(fma_f(x.at(j) - g.ref, c, g.k));
  }
  RowVec<DT> y;
  y.set(d);
  if (g.sign)
#pragma unroll
    for (int i = 0; i < RowVec<DT>::WORDS; ++i) y.w[i] ^= DT == STRIM_DTYPE_BF16 ? g.sign : 0x80000000u;
  if (g.dead)
#pragma unroll
    for (int i = 0; i < RowVec<DT>::WORDS; ++i) y.w[i] = 0;
  return y;
}
// The gradients of the wave's own alternatives among its tokens, a lane each, over what the wave stored there
// before: a wave's stores to one address keep their order. id -1: none.
template <int DT>
__device__ __forceinline__ void grad_alternatives(char* out, const GradRow& g, float c, const int (&id)[2],
                                                  const float (&x)[2], const float (&p)[2]) {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if (g.dead) return;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (id[i] >= 0) {
      const float f = g.in * hw_exp2(fma_f(x[i] - g.top, c, g.kq)) - p[i];
      if constexpr (DT == STRIM_DTYPE_BF16) ((uint16_t*)out)[id[i]] = __builtin_bit_cast(uint16_t, (__bf16)f);
      else ((float*)out)[id[i]] = f;
    }
}

// The row's alternatives for the gradient, each id once: what the waves read, in LDS or from memory.
struct GradList {
  int id[DI_M];
  float x[DI_M], p[DI_M];  // its logit, and w / T p_m
  int repeats;             // whether an id stands twice
};
// What k_distill_join leaves for the gradient of a step.
struct GradRecord {
  GradRow row;
  GradList list;
};
// Looks for repeated ids, all threads: entry e against a part of those before it. (Two barriers' worth:
// the caller's before reading l.repeats.)
template <int T>
__device__ __forceinline__ void find_repeats(GradList& l, const Alternatives& o) {
  if (threadIdx.x < WAVE) {
    l.id[threadIdx.x] = o.id[0];
    l.id[threadIdx.x + WAVE] = o.id[1];
    if (threadIdx.x == 0) l.repeats = 0;
  }
  __syncthreads();
  constexpr int SEG = DI_M * DI_M / T;
  const int e = threadIdx.x % DI_M, from = (int)threadIdx.x / DI_M * SEG, id = l.id[e];
  bool twice = false;
#pragma unroll 4
  for (int j = from; j < from + SEG; ++j) twice |= j < e && l.id[j] == id;
  if (twice && id >= 0) l.repeats = 1;
}
// The wave's entries as GradList has them, each id once. x: their logits.
__device__ __forceinline__ void list_out(GradList& l, const Alternatives& o, const Teacher& t, int M, double w,
                                         const float (&x)[2], bool (&first)[2], bool repeats) {
  const int lane = threadIdx.x & (WAVE - 1);
  float p[2] = {t.p[0], t.p[1]};
  if (repeats) merge_repeats(o, M, first, p);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l.id[lane + i * WAVE] = first[i] ? o.id[i] : -1;
    l.x[lane + i * WAVE] = x[i];
    l.p[lane + i * WAVE] = (float)(w * p[i]);
  }
}

struct DistillParts {
  int32_t parts, tiles;  // parts of a row; tiles of a part
  RowStat* part;         // [N][parts]
  GradRecord* record;    // a step's: [N]
};

// The tokens' statistic of a part of a row; TAIL: without the alternatives'.
template <int DT, bool TAIL>
__global__ __launch_bounds__(DI_T) void k_distill_stat(const DistillArgs a, const DistillParts q) {
  __shared__ RowStat s_stat[DI_T / WAVE];
  const int64_t r = blockIdx.x / q.parts;
  const int p = blockIdx.x - (int)r * q.parts, lane = threadIdx.x & (WAVE - 1), wave = wave_id();
  const char* row = (const char*)a.logits + r * a.stride * RowVec<DT>::SIZE;
  const float c = LOG2E / a.T;
  const int t0 = p * q.tiles * DI_TILE, t1 = min(a.V, t0 + q.tiles * DI_TILE);
  RowVec<DT> next[DI_U];
  auto request = [&](int t) {
#pragma unroll
    for (int u = 0; u < DI_U; ++u) {
      const int w0 = t + 8 * WAVE * (u * (DI_T / WAVE) + wave);
      if (t + DI_TILE <= a.V) next[u].template load<true>(row, w0, lane);
      else next[u].load_to(row, w0, lane, a.V);
    }
  };
  request(t0);
  Alternatives o;
  if constexpr (TAIL) o = alternatives_of(a, r);
  RowStat st{-INFINITY, 0.0f, 0.0f};
  for (int t = t0; t < t1; t += DI_TILE) {
    float x[8 * DI_U];
#pragma unroll
    for (int u = 0; u < DI_U; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[8 * u + j] = next[u].at(j);
    if (t + DI_TILE < t1) request(t + DI_TILE);
    if constexpr (TAIL)
#pragma unroll
      for (int u = 0; u < DI_U; ++u)
        each_hit<DT>(o.id, t + 8 * WAVE * (u * (DI_T / WAVE) + wave), [&](int at, int e, int, int) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (lane == at && j == e) x[8 * u + j] = -INFINITY;
        });
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8 * DI_U; ++j) mx = fmaxf(mx, x[j]);
    stat_add<8 * DI_U, false>(st, x, mx, c);
  }
  stat_wave(st, c);
  if (lane == 0) s_stat[threadIdx.x / WAVE] = st;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < DI_T / WAVE; ++i) stat_merge(st, s_stat[i], c);
    q.part[r * q.parts + p] = st;
  }
}

// The rows' results; a wave a row. STEP: and what the gradient takes of them.
template <int DT, bool STEP>
__global__ __launch_bounds__(WAVE) void k_distill_join(const DistillArgs a, const DistillParts q) {
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x;
  const float c = LOG2E / a.T;
  const char* row = (const char*)a.logits + r * a.stride * RowVec<DT>::SIZE;
  const Alternatives o = alternatives_of(a, r);
  RowStat st{-INFINITY, 0.0f, 0.0f};
  for (int p = lane; p < q.parts; p += WAVE) stat_merge(st, q.part[r * q.parts + p], c);
  const double w = STEP ? (double)a.weights[r] / a.T : 0.0;
  float x[2], merged[2] = {0.0f, 0.0f};
  bool first[2] = {true, true};
#pragma unroll
  for (int i = 0; i < 2; ++i) x[i] = o.any && o.id[i] >= 0 ? token_at<DT>(row, o.id[i]) : -INFINITY;
  stat_wave(st, c);
  stat_exact(st, c);
  const Teacher t = teacher_of(o, a.tail);
  if (a.tail || STEP) {
#pragma unroll
    for (int i = 0; i < 2; ++i) merged[i] = t.p[i];
    merge_repeats(o, a.M, first, merged);
  }
  RowNumbers n{};
  if (o.any) n = numbers_of(o, t, first, x, st, a.T, a.tail);
  if constexpr (STEP) {
    GradRecord* rec = q.record + r;
    const GradRow g = grad_row(o.any, t, n, w, c);
    if (lane == 0) rec->row = g;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      rec->list.id[lane + i * WAVE] = first[i] ? o.id[i] : -1;
      rec->list.x[lane + i * WAVE] = x[i];
      rec->list.p[lane + i * WAVE] = (float)(w * merged[i]);
    }
  }
  if (lane != 0) return;
  const float loss = (float)n.loss;
  a.loss[r] = loss;
  if (a.out_lse) a.out_lse[r] = (float)(n.top / a.T + n.ls);
  if (a.out_log_rest) a.out_log_rest[r] = (float)n.log_rest;
  if (a.status)
    a.status[r] = !o.known ? STRIM_EINVAL : fabsf(loss) < INFINITY ? STRIM_OK : STRIM_ENONFINITE;
}

// A part of a row's gradient: from its lse and log q_rest, or (STEP) from its record.
template <int DT, bool STEP>
__global__ __launch_bounds__(DI_T) void k_distill_grad(const DistillArgs a, const DistillParts q) {
  __shared__ GradList s_list;
  __shared__ GradRow s_grad;
  const int64_t r = blockIdx.x / q.parts;
  const int p = blockIdx.x - (int)r * q.parts, lane = threadIdx.x & (WAVE - 1), wave = wave_id();
  const char* row = (const char*)a.logits + r * a.stride * RowVec<DT>::SIZE;
  char* out = (char*)a.d_logits + r * a.d_stride * RowVec<DT>::SIZE;
  const float c = LOG2E / a.T;
  const int t0 = p * q.tiles * DI_TILE, t1 = min(a.V, t0 + q.tiles * DI_TILE);
  RowVec<DT> next[DI_U];
  auto request = [&](int t) {
#pragma unroll
    for (int u = 0; u < DI_U; ++u)
      next[u].template load_to<false, true>(row, t + 8 * WAVE * (u * (DI_T / WAVE) + wave), lane, a.V);
  };
  request(t0);
  const GradList* list = &s_list;
  GradRow g;
  if constexpr (STEP) {
    list = &q.record[r].list;
    g = q.record[r].row;
  } else {
    const Alternatives o = alternatives_of(a, r);
    find_repeats<DI_T>(s_list, o);
    __syncthreads();
    if (wave == 0) {
      const Teacher t = teacher_of(o, a.tail);
      const double w = (double)a.weights[r] / a.T;
      bool first[2] = {o.id[0] >= 0, o.id[1] >= 0};
      float x[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) x[i] = o.any && o.id[i] >= 0 ? token_at<DT>(row, o.id[i]) : -INFINITY;
      list_out(s_list, o, t, a.M, w, x, first, s_list.repeats != 0);
      g = grad_row(o.any, t, numbers_from(a.lse[r], a.tail ? (double)a.log_rest[r] : 0.0, a.tail, a.T), w, c);
      if (lane == 0) s_grad = g;
    }
    __syncthreads();
    g = s_grad;
  }
  // the wave's own alternatives
  int id[2];
  float x[2], less[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    id[i] = list->id[lane + i * WAVE];
    x[i] = list->x[lane + i * WAVE];
    less[i] = list->p[lane + i * WAVE];
    if (id[i] < t0 || id[i] >= t1 || id[i] / (8 * WAVE) % (DI_T / WAVE) != wave) id[i] = -1;
  }
  for (int s = t0; s < t1; s += DI_TILE) {
    RowVec<DT> now[DI_U];
#pragma unroll
    for (int u = 0; u < DI_U; ++u) now[u] = next[u];
    if (s + DI_TILE < t1) request(s + DI_TILE);
#pragma unroll
    for (int u = 0; u < DI_U; ++u) {
      const int w0 = s + 8 * WAVE * (u * (DI_T / WAVE) + wave);
      if (w0 >= a.V) break;
      grad_of<DT>(now[u], g, c).store_to(out, w0, lane, a.V, a.stream);
    }
  }
  grad_alternatives<DT>(out, g, c, id, x, less);
}

// A row whole: NV vectors of eight tokens a thread in registers, KEEP more in LDS (one workgroup a CU, or two; bf16,
// V = 151,936, N = 4,096 571 us without, 547 with; float32, N = 1,024 297 and 283); what is past them is read again for
// the gradient.
template <int DT, int T, int NV, bool TAIL>
__global__ __launch_bounds__(T) void k_distill_step(const DistillArgs a) {
  constexpr int NWAVES = T / WAVE, WORDS = RowVec<DT>::WORDS;
  constexpr int KEEP = NV <= 4 ? 0 : (T == 512 ? 72 : 136) * 1024 / (T * WORDS * 4);
  __shared__ uint32_t s_keep[KEEP > 0 ? KEEP : 1][KEEP > 0 ? WORDS / 4 : 1][KEEP > 0 ? 4 * T : 4];
  auto keep = [&](int k, RowVec<DT>& q) -> void {
    if constexpr (KEEP > 0)
#pragma unroll
      for (int i = 0; i < WORDS / 4; ++i)
        *(ru32x4*)&s_keep[k][i][4 * threadIdx.x] = ru32x4{q.w[4 * i], q.w[4 * i + 1], q.w[4 * i + 2], q.w[4 * i + 3]};
  };
  __shared__ RowStat s_stat[NWAVES];
  __shared__ GradList s_list;
  __shared__ GradRow s_grad;
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x & (WAVE - 1), wave = wave_id();
  const char* row = (const char*)a.logits + r * a.stride * RowVec<DT>::SIZE;
  char* out = (char*)a.d_logits + r * a.d_stride * RowVec<DT>::SIZE;
  const float c = LOG2E / a.T;
  RowVec<DT> x[NV];
#pragma unroll
  for (int u = 0; u < NV; ++u) x[u].template load_to<false, true>(row, 8 * WAVE * (u * NWAVES + wave), lane, a.V);
  const Alternatives o = alternatives_of(a, r);
  find_repeats<T>(s_list, o);
  // the vectors among which the wave's alternatives are
  uint64_t hits = 0;
  if constexpr (TAIL)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      for (uint64_t b = __ballot(o.id[i] >= 0 && (o.id[i] / (8 * WAVE)) % NWAVES == wave); b; b &= b - 1)
        hits |= 1ull << min(63, rl_i(o.id[i], __builtin_ctzll(b)) / (8 * T));
  RowStat st{-INFINITY, 0.0f, 0.0f};
  // two vectors at a time
  auto add = [&](const RowVec<DT>& q0, const RowVec<DT>& q1, int w0, int w1, bool hit0, bool hit1) {
    float f[16], mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[j] = q0.at(j);
      f[8 + j] = q1.at(j);
    }
    if constexpr (TAIL) {
      if (hit0) without_hits<DT>(*(float(*)[8])&f[0], o.id, w0);
      if (hit1) without_hits<DT>(*(float(*)[8])&f[8], o.id, w1);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) mx = fmaxf(mx, f[j]);
    stat_add<16, false>(st, f, mx, c);
  };
  RowVec<DT> none;
#pragma unroll
  for (int i = 0; i < RowVec<DT>::WORDS; ++i) none.w[i] = DT == STRIM_DTYPE_BF16 ? 0xFF80FF80u : NINF_BITS;
#pragma unroll
  for (int u = 0; u < NV; u += 2) {
    const int w0 = 8 * WAVE * (u * NWAVES + wave), w1 = w0 + 8 * T;
    add(x[u], u + 1 < NV ? x[u + 1] : none, w0, w1, (hits >> u) & 1u, u + 1 < NV && ((hits >> (u + 1)) & 1u));
    x[u].renew();  // (568 bytes a lane spilled without)
    if (u + 1 < NV) x[u + 1].renew();
  }
  for (int v0 = 8 * NV * T; v0 < a.V; v0 += 16 * T) {
    const int w0 = v0 + 8 * WAVE * wave, w1 = w0 + 8 * T;
    RowVec<DT> q0, q1;
    q0.load_to(row, w0, lane, a.V);
    q1.load_to(row, w1, lane, a.V);
    add(q0, q1, w0, w1, true, true);
    const int k = v0 / (8 * T) - NV;
    if (k < KEEP) keep(k, q0);
    if (k + 1 < KEEP) keep(k + 1, q1);
  }
  stat_wave(st, c);
  if (lane == 0) s_stat[wave] = st;
  __syncthreads();
  if (wave == 0) {
    st = lane < NWAVES ? s_stat[lane] : RowStat{-INFINITY, 0.0f, 0.0f};
    stat_wave(st, c);
    stat_exact(st, c);
    const Teacher t = teacher_of(o, TAIL);
    const double w = (double)a.weights[r] / a.T;
    bool first[2] = {o.id[0] >= 0, o.id[1] >= 0};
    float xa[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) xa[i] = o.any && o.id[i] >= 0 ? token_at<DT>(row, o.id[i]) : -INFINITY;
    list_out(s_list, o, t, a.M, w, xa, first, s_list.repeats != 0);
    RowNumbers n{};
    if (o.any) n = numbers_of(o, t, first, xa, st, a.T, TAIL);
    const GradRow g = grad_row(o.any, t, n, w, c);
    if (lane == 0) {
      s_grad = g;
      const float loss = (float)n.loss;
      a.loss[r] = loss;
      if (a.status)
        a.status[r] = !o.known ? STRIM_EINVAL : fabsf(loss) < INFINITY ? STRIM_OK : STRIM_ENONFINITE;
    }
  }
  __syncthreads();
  const GradRow g = s_grad;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int w0 = 8 * WAVE * (u * NWAVES + wave);
    if (w0 < a.V) grad_of<DT>(x[u], g, c).store_to(out, w0, lane, a.V, a.stream);
  }
  int k = 0;
  for (int w0 = 8 * (NV * T + WAVE * wave); w0 < a.V; w0 += 8 * T, ++k) {
    RowVec<DT> q;
    if (k < KEEP) {
#pragma unroll
      for (int i = 0; i < (KEEP > 0 ? WORDS / 4 : 0); ++i) {
        const ru32x4 v = *(const ru32x4*)&s_keep[k][i][4 * threadIdx.x];
#pragma unroll
        for (int j = 0; j < 4; ++j) q.w[4 * i + j] = v[j];
      }
    } else {
      q.load_to(row, w0, lane, a.V);
    }
    grad_of<DT>(q, g, c).store_to(out, w0, lane, a.V, a.stream);
  }
  int id[2];
  float xa[2], less[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    id[i] = s_list.id[lane + i * WAVE];
    xa[i] = s_list.x[lane + i * WAVE];
    less[i] = s_list.p[lane + i * WAVE];
    if (id[i] >= 0 && id[i] / (8 * WAVE) % NWAVES != wave) id[i] = -1;
  }
  grad_alternatives<DT>(out, g, c, id, xa, less);
}

// (a factor of 1, what the last step of a backward pass usually has, costs no pass over the data; another a pass of
// one element a lane: N = 4,096, V = 151,936 in bf16 854 us, 2.9 TB/s)
template <int DT>
__global__ __launch_bounds__(DI_T) void k_distill_scale(char* data, int64_t n, const float* factor) {
  const float f = *factor;
  if (f == 1.0f) return;
  for (int64_t i = (int64_t)blockIdx.x * DI_T + threadIdx.x; i < n; i += (int64_t)gridDim.x * DI_T) {
    if constexpr (DT == STRIM_DTYPE_BF16) {
      uint16_t* p = (uint16_t*)data + i;
      *p = __builtin_bit_cast(uint16_t, (__bf16)(bf16_to_f32(*p) * f));
    } else {
      ((float*)data)[i] *= f;
    }
  }
}

int64_t up16(int64_t b) { return (b + 15) & ~(int64_t)15; }
int64_t ceil_of(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Parts of a row: a round of workgroups over the chip (eight a CU), one a row where there are that many rows;
// float32 rows, whose kernels hold fewer, in two rounds (N = 500, V = 50,021: 29.0 -> 26.4 us).
DistillParts distill_parts(int N, int V, bool bf16) {
  DistillParts q{};
  const int64_t tiles = ceil_of(V, DI_TILE), each = ceil_of((int64_t)N * tiles, bf16 ? 2048 : 4096);
  q.tiles = (int32_t)(each > tiles ? tiles : each);
  q.parts = (int32_t)ceil_of(tiles, q.tiles);
  return q;
}
// Whether a step keeps each row in a workgroup: always where four vectors a thread hold it, else from half a round
// of rows on. Replayed steps of N = 1, 64, 96, 127, 200, whole and in parts, us:
//   bf16     V = 32,768   8.9, 10.4, 10.4, 11.2, 12.3   13.5, 14.8, 15.8, 16.1, 18.5
//            V = 40,000   18, 19, 20, 20, 21            14, 16, 16, 17, 20
//            V = 100,003  19, 28, 29, 30, 33            14, 20, 22, 27, 36
//            V = 151,936  21, 27, 28, 29, 33            13, 21, 26, 33, 43
//   float32  V = 40,000   13, 15, 16, 18, 21            13, 17, 18, 20, 24
//            V = 151,936  23, 32, 34, 38, 49            13, 29, 38, 48, 66
// (float32 rows of 40,000 and 65,536 tokens would be as fast or faster whole from one row on.)
bool whole_rows(int N, int V) { return N >= 128 || V <= 8 * 1024 * 4; }

template <class F>
void with_dtype(bool bf16, F f) {
  if (bf16) f(std::integral_constant<int, STRIM_DTYPE_BF16>{});
  else f(std::integral_constant<int, STRIM_DTYPE_F32>{});
}

template <int DT, bool TAIL>
void launch_whole(const DistillArgs& a, hipStream_t st) {
  constexpr int MOST = 1 << 21;  // (a launch has fewer than 2^32 threads)
  for (int r0 = 0; r0 < a.N; r0 += MOST) {
    DistillArgs b = a;
    const int64_t at = r0;
    b.N = a.N - r0 < MOST ? a.N - r0 : MOST;
    b.logits = (const char*)a.logits + at * a.stride * RowVec<DT>::SIZE;
    b.d_logits = (char*)a.d_logits + at * a.d_stride * RowVec<DT>::SIZE;
    b.ids = a.ids + at * a.M;
    b.logprobs = a.logprobs + at * a.M;
    b.weights = a.weights + at;
    b.loss = a.loss + at;
    if (a.status) b.status = a.status + at;
    auto go = [&](auto kernel, int threads) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)b.N), dim3(threads), 0, st, b);
    };
    // The whole row in registers, or, where there are rows for it, half of it with two workgroups a CU, one
    // of which reads while the other writes (V = 151,936, 2.5 GB read and written, N = 4,096: 587 -> 571 us, with KEEP 547; N =
    // 128 35 -> 43; V = 248,320, N = 1,024, where only a third would be held: 254 -> 286).
    if (a.V <= 8 * 256 * 4) {
      go(k_distill_step<DT, 256, 4, TAIL>, 256);
    } else if (a.V <= 8 * 1024 * 4) {
      go(k_distill_step<DT, 1024, 4, TAIL>, 1024);
    } else if constexpr (DT == STRIM_DTYPE_BF16) {
      if (a.N > 256 && a.V <= 8 * 1024 * 19) go(k_distill_step<DT, 512, 19, TAIL>, 512);
      else go(k_distill_step<DT, 1024, 19, TAIL>, 1024);
    } else {
      go(k_distill_step<DT, 1024, 9, TAIL>, 1024);
    }
  }
}

}  // namespace

int64_t distill_workspace(int N, int V, int M, bool step) {
  (void)M;
  if (step && whole_rows(N, V)) return 0;
  // (the parts of the type that has more)
  const int64_t parts = distill_parts(N, V, true).parts, most = distill_parts(N, V, false).parts;
  return up16((int64_t)N * (parts > most ? parts : most) * (int64_t)sizeof(RowStat)) +
         (step ? (int64_t)N * (int64_t)sizeof(GradRecord) : 0);
}

hipError_t launch_distill(const DistillArgs& given, bool bf16, bool loss, bool grad, void* workspace,
                          hipStream_t st) {
  DistillArgs a = given;
  a.stream = grad && (int64_t)a.N * a.V * (bf16 ? 2 : 4) > ROWS_CACHED;
  const bool step = loss && grad;
  if (step && whole_rows(a.N, a.V)) {
    with_dtype(bf16, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      a.tail ? launch_whole<DT, true>(a, st) : launch_whole<DT, false>(a, st);
    });
    return hipGetLastError();
  }
  DistillParts q = distill_parts(a.N, a.V, bf16);
  if (loss) {
    q.record = (GradRecord*)workspace;
    q.part = (RowStat*)(step ? (void*)(q.record + a.N) : workspace);
  }
  const dim3 grid((unsigned)((int64_t)a.N * q.parts)), threads(DI_T), rows((unsigned)a.N);
  with_dtype(bf16, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (loss) {
      if (a.tail) hipLaunchKernelGGL((k_distill_stat<DT, true>), grid, threads, 0, st, a, q);
      else hipLaunchKernelGGL((k_distill_stat<DT, false>), grid, threads, 0, st, a, q);
      if (step) hipLaunchKernelGGL((k_distill_join<DT, true>), rows, dim3(WAVE), 0, st, a, q);
      else hipLaunchKernelGGL((k_distill_join<DT, false>), rows, dim3(WAVE), 0, st, a, q);
    }
    if (step) hipLaunchKernelGGL((k_distill_grad<DT, true>), grid, threads, 0, st, a, q);
    else if (grad) hipLaunchKernelGGL((k_distill_grad<DT, false>), grid, threads, 0, st, a, q);
  });
  return hipGetLastError();
}

hipError_t launch_distill_scale(void* data, bool bf16, int64_t n, const float* factor, hipStream_t st) {
  const int64_t blocks = ceil_of(n, DI_T);
  with_dtype(bf16, [&](auto dt) {
    hipLaunchKernelGGL(k_distill_scale<decltype(dt)::value>, dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(DI_T), 0,
                       st, (char*)data, n, factor);
  });
  return hipGetLastError();
}

}  // namespace strim
