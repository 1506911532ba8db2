// top.hpp — the first M tokens of a row in token order (logit descending, then id), M <= TOP_MAX, by one
// workgroup of TOP_T threads that meets the row a tile at a time.
//
// Each thread keeps the largest logit it has met. The M-th largest of the threads' maxima is no larger
// than the M-th largest logit met so far, and hardly smaller: with 256 threads and M = 64 about 74
// logits reach it. So tokens that reach this threshold are appended to a list in LDS, the threshold is
// raised after tiles 1, 4, 16, ... (between two of them about 3 M tokens are appended), and at the end
// the list is cut at the last threshold and ordered. Ids ascend from tile to tile: once M tokens have
// reached a threshold, a later one that only equals it is past the M-th.
#pragma once

#include "common.hpp"

namespace strim {

constexpr int TOP_T = 256;
constexpr int TOP_MAX = STRIM_SCORE_MAX_LIST;
constexpr int TOP_STEP = 2048;             // tokens appended at most between two looks at the list's length
constexpr int TOP_CAP = TOP_STEP + TOP_T;  // list: what was there when it was last cut, and a step
static_assert(TOP_MAX <= TOP_T, "a list that was cut leaves room for a step");
constexpr uint32_t TOP_ALL = 0xFF7FFFFFu;  // fkey_desc of the lowest finite value: every token above -inf

struct TopList {
  uint64_t key[TOP_CAP];  // ckey, in no order
  uint32_t best[TOP_T];   // fkey_desc of the threads' maxima
  int n;
  int added[3];           // entries that a tile appended: this one's, the last one's, the next one's
  int part[2][TOP_T / WAVE];
  uint64_t bound[2];
};

// The threshold from the threads' maxima (as fkey_desc keys: larger logits have smaller ones): a key that
// M of them reach, the least one to 2^-15 of the keys' range; TOP_ALL where fewer than M have a finite
// logit. Every wave finds it by itself, halving the range.
__device__ __forceinline__ uint32_t top_threshold(TopList& l, uint32_t mine, int M) {
  l.best[threadIdx.x] = mine;
  __syncthreads();
  uint32_t b[TOP_T / WAVE];
#pragma unroll
  for (int i = 0; i < TOP_T / WAVE; ++i) b[i] = l.best[i * WAVE + (threadIdx.x & (WAVE - 1))];
  auto reach = [&](uint32_t t) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < TOP_T / WAVE; ++i) n += __popcll(__ballot(b[i] <= t));
    return n;
  };
  if (reach(TOP_ALL) < M) return TOP_ALL;
  uint32_t lo = 0, hi = TOP_ALL;  // reach(hi) >= M; the result is in (lo, hi]
  while (hi - lo > 0x8000u) {     // (17 steps)
    const uint32_t mid = lo + (hi - lo) / 2;
    if (reach(mid) >= M) hi = mid;
    else lo = mid;
  }
  return hi;
}

// Cuts the list's n keys to those that are at most `limit` (their order is lost). All threads; returns the
// new length.
__device__ __forceinline__ int top_cut(TopList& l, int n, uint64_t limit) {
  constexpr int Q = TOP_CAP / TOP_T;
  uint64_t k[Q];
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const int at = i * TOP_T + (int)threadIdx.x;
    k[i] = at < n ? l.key[at] : ~0ull;
  }
  __syncthreads();
  if (threadIdx.x == 0) l.n = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < Q; ++i)
    if (i * TOP_T < n && k[i] != ~0ull && k[i] <= limit) l.key[atomicAdd(&l.n, 1)] = k[i];
  __syncthreads();
  n = l.n;
  __syncthreads();
  return n;
}

// The M-th smallest of the list's n > M keys (they all differ), by halving the range between the least and
// the largest: a count of the workgroup's keys a step.
__device__ __noinline__ uint64_t top_select(lds_t<TopList>* lp, int n, int M) {
  TopList& l = *(TopList*)lp;
  n = __builtin_amdgcn_readfirstlane(n);
  M = __builtin_amdgcn_readfirstlane(M);
  constexpr int Q = TOP_CAP / TOP_T;
  uint64_t k[Q];
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const int at = i * TOP_T + (int)threadIdx.x;
    k[i] = at < n ? l.key[at] : ~0ull;
  }
  uint64_t lo = 0, hi = (uint64_t)TOP_ALL << 32 | 0xFFFFFFFFu;  // count(hi) >= M > count(lo)
  for (int step = 0; hi - lo > 1; ++step) {
    const uint64_t mid = lo + (hi - lo) / 2;
    int c = 0;
#pragma unroll
    for (int i = 0; i < Q; ++i) c += __popcll(__ballot(k[i] <= mid));
    if ((threadIdx.x & (WAVE - 1)) == 0) l.part[step & 1][threadIdx.x / WAVE] = c;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int i = 0; i < TOP_T / WAVE; ++i) all += l.part[step & 1][i];
    if (__builtin_amdgcn_readfirstlane(all) >= M) hi = mid;
    else lo = mid;
  }
  __syncthreads();
  return hi;
}

// The list cut to its first M keys (still in no order); `limit` is lowered to below the last one's logit, if
// there are M: tokens that come later have larger ids.
__device__ __forceinline__ int top_reduce(TopList& l, int n, int M, uint32_t& limit) {
  if (n <= M) return n;
  const uint64_t last = top_select((lds_t<TopList>*)&l, n, M);
  limit = min(limit, (uint32_t)(last >> 32) - 1u);
  return top_cut(l, n, last);
}

// The workgroup's view of the list while the row goes by.
struct TopRun {
  int held, tile;   // entries; tiles met
  uint32_t limit;   // tokens whose fkey_desc is at most this are appended
  int M;

  __device__ __forceinline__ void init(TopList& l, int m) {
    held = tile = 0;
    limit = TOP_ALL;
    M = m;
    if (threadIdx.x < 3) l.added[threadIdx.x] = 0;
    __syncthreads();
  }

  // A tile of U slots of TOP_STEP tokens, eight a thread: x[8 u ..] are the thread's of slot u, from id
  // first + u TOP_STEP on; mx is their maximum, most the largest that the thread has met.
  template <int U>
  __device__ __forceinline__ void add(TopList& l, const float (&x)[8 * U], float mx, float most, int first) {
    // (tiles 0, 3, 15, 63, ...: each time the list's length has grown by 3 M or so)
    const bool raise = tile == 0 || (((tile + 1) & tile) == 0 && ((tile + 1) & 0x55555554) != 0);
    uint32_t raised = 0;
    if (raise) {
      raised = top_threshold(l, fkey_desc(most), M);
      limit = min(limit, raised);
    }
    float floor = fkey_desc_inv(limit);
    int* added = &l.added[tile % 3];
    if (threadIdx.x == 0) l.added[(tile + 1) % 3] = 0;
    if (mx >= floor)
#pragma unroll
      for (int j = 0; j < 8 * U; ++j)
        if (x[j] >= floor) {
          const int at = held + atomicAdd(added, 1);
          if (at < TOP_CAP) l.key[at] = ckey(x[j], first + (j >> 3) * TOP_STEP + (j & 7));
        }
    __syncthreads();
    const int more = __builtin_amdgcn_readfirstlane(*added);
    if (held + more > TOP_CAP) {
      // too many at once (ties, or a run of large ones): slot by slot, the list cut in between
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (held > TOP_T) held = top_reduce(l, held, M, limit);
        floor = fkey_desc_inv(limit);
        __syncthreads();
        if (threadIdx.x == 0) l.n = held;
        __syncthreads();
#pragma unroll
        for (int j = 8 * u; j < 8 * u + 8; ++j)
          if (x[j] >= floor) l.key[atomicAdd(&l.n, 1)] = ckey(x[j], first + u * TOP_STEP + (j & 7));
        __syncthreads();
        held = __builtin_amdgcn_readfirstlane(l.n);
      }
      __syncthreads();
    } else {
      held += more;
    }
    // M tokens have reached the raised threshold: later ones that only equal it are past them
    if (raise && raised != TOP_ALL) limit = min(limit, raised - 1u);
    ++tile;
  }

  // The list without what the threads' maxima show to be past the M-th.
  __device__ __forceinline__ void trim(TopList& l, float most) {
    if (held <= M || tile == 1) return;  // (after one tile the list is at its threshold)
    const uint32_t t = top_threshold(l, fkey_desc(most), M);
    held = top_cut(l, held, (uint64_t)t << 32 | 0xFFFFFFFFu);
  }
};

// put(place, key) for the list's first M keys; a key's place is the number of smaller ones.
template <class F>
__device__ __forceinline__ void top_order(TopList& l, int n, int M, F put) {
  uint32_t unused = 0;
  if (n > 2 * TOP_T) n = top_reduce(l, n, M, unused);
  for (int at = threadIdx.x; at < n; at += TOP_T) {
    const uint64_t k = l.key[at];
    int r = 0;
    for (int j = 0; j < n; ++j) r += l.key[j] < k ? 1 : 0;
    if (r < M) put(r, k);
  }
}

}  // namespace strim
