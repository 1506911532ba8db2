// top.hpp — the first M tokens of a row in token order (logit descending, then id), M <= TOP_MAX, by one
// workgroup of TOP_T threads that meets the row a tile at a time.
//
// Each thread keeps the largest logit it has met. The M-th largest of the threads' maxima is no larger
// than the M-th largest logit met so far, and hardly smaller: with 256 threads and M = 64 about 74
// logits reach it. So tokens that reach this threshold are appended to a list in LDS, the threshold is
// raised after tiles 1, 2, 4, 8, ... (between two of them about M tokens are appended), and at the end
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

// A list entry as it is appended: the logit's bits and the id, made into a ckey when the list is cut or
// ordered (seven instructions that most entries need once, off the tokens' path).
__device__ __forceinline__ uint64_t top_entry(float x, int id) {
  return (uint64_t)__float_as_uint(x) << 32 | (uint32_t)id;
}
__device__ __forceinline__ uint64_t top_key(uint64_t entry) {
  return ckey(__uint_as_float((uint32_t)(entry >> 32)), (int32_t)(uint32_t)entry);
}

constexpr uint64_t TOP_NONE = 0xFF80000000000000ull;  // an entry of -inf: no token

struct TopList {
  uint64_t e[TOP_CAP];   // entries, in no order
  uint32_t best[TOP_T];  // fkey_desc of the threads' maxima
  uint32_t limit;
  int n;
  int added[3];          // entries that a tile appended: this one's, the last one's, the next one's
  int part[2][TOP_T / WAVE];
};

// A threshold from the threads' maxima (as fkey_desc keys: larger logits have smaller ones), no larger than
// `hi`: a key that M of them reach, the least one to 2^15 keys; `hi` where fewer than M reach that. One wave
// halves the range (`by`: which), the others wait.
__device__ __forceinline__ uint32_t top_threshold(TopList& l, uint32_t mine, uint32_t hi, int M, int by) {
  l.best[threadIdx.x] = mine;
  __syncthreads();
  if (wave_id() == by) {
    uint32_t b[TOP_T / WAVE];
#pragma unroll
    for (int i = 0; i < TOP_T / WAVE; ++i) b[i] = l.best[i * WAVE + (threadIdx.x & (WAVE - 1))];
    auto reach = [&](uint32_t t) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < TOP_T / WAVE; ++i) n += __popcll(__ballot(b[i] <= t));
      return n;
    };
    hi = __builtin_amdgcn_readfirstlane(hi);
    if (reach(hi) >= M) {
      // reach(hi) >= M throughout; the result is in (lo, hi], as a rule within three octaves of the old one
      uint32_t lo = hi > 0x02000000u ? hi - 0x02000000u : 0u;
      if (reach(lo) >= M) {
        hi = lo;
        lo = 0;
      }
      while (hi - lo > 0x8000u) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (reach(mid) >= M) hi = mid;
        else lo = mid;
      }
    }
    if ((threadIdx.x & (WAVE - 1)) == 0) l.limit = hi;
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(l.limit);
}

// Cuts the list's n entries to those whose key is at most `limit` (their order is lost). All threads; returns
// the new length.
__device__ __forceinline__ int top_cut(TopList& l, int n, uint64_t limit) {
  constexpr int Q = TOP_CAP / TOP_T;
  uint64_t e[Q];
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const int at = i * TOP_T + (int)threadIdx.x;
    e[i] = at < n ? l.e[at] : 0;
  }
  __syncthreads();
  if (threadIdx.x == 0) l.n = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < Q; ++i)
    if (i * TOP_T + (int)threadIdx.x < n && top_key(e[i]) <= limit) l.e[atomicAdd(&l.n, 1)] = e[i];
  __syncthreads();
  n = __builtin_amdgcn_readfirstlane(l.n);
  __syncthreads();
  return n;
}

// The M-th smallest of the list's n > M keys (they all differ), by halving the range between the least and
// the largest: a count of the workgroup's keys a step.
__device__ __forceinline__ uint64_t top_select(TopList& l, int n, int M) {
  constexpr int Q = TOP_CAP / TOP_T;
  uint64_t k[Q];
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const int at = i * TOP_T + (int)threadIdx.x;
    k[i] = at < n ? top_key(l.e[at]) : ~0ull;
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

// The list cut to its first M entries (still in no order); `limit` is lowered to below the last one's logit:
// tokens that come later have larger ids.
__device__ __forceinline__ int top_reduce(TopList& l, int n, int M, uint32_t& limit) {
  if (n <= M) return n;
  const uint64_t last = top_select(l, n, M);
  limit = min(limit, (uint32_t)(last >> 32) - 1u);
  return top_cut(l, n, last);
}

// The workgroup's view of the list while the row goes by.
struct TopRun {
  int held, tile;   // entries; tiles met
  uint32_t limit;   // tokens whose fkey_desc is at most this are appended
  int M, by;
  uint32_t before;  // the limit before this tile

  __device__ __forceinline__ void init(TopList& l, int m) {
    by = blockIdx.x % (TOP_T / WAVE);
    held = tile = 0;
    limit = TOP_ALL;
    M = m;
    if (threadIdx.x < 3) l.added[threadIdx.x] = 0;
    __syncthreads();
  }

  // A tile of U slots of TOP_STEP tokens, eight a thread: x[8 u ..] are the thread's of slot u, with ids
  // first + u TOP_STEP + step(j); mv[u] is their maximum, `most` the largest that the thread has met. False where
  // more were to be appended than the list holds: the tile is then given to top_slots.
  template <int U, class S>
  __device__ __forceinline__ bool add(TopList& l, const float (&x)[8 * U], const float (&mv)[U], float most, int first,
                                      S step) {
    const bool raise = ((tile + 1) & tile) == 0;
    before = limit;
    if (raise) limit = top_threshold(l, fkey_desc(most), limit, M, by);
    const float floor = fkey_desc_inv(limit);
    int* added = &l.added[tile % 3];
    if (threadIdx.x == 0) l.added[(tile + 1) % 3] = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (__ballot(mv[u] >= floor)) {
        // one atomic for the wave's tokens: its lanes' places follow from the ballots
        uint64_t m[8];
        int n = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          m[j] = __ballot(x[8 * u + j] >= floor);
          n += __popcll(m[j]);
        }
        int at = 0;
        if ((threadIdx.x & (WAVE - 1)) == 0) at = atomicAdd(added, n);
        at = held + __builtin_amdgcn_readfirstlane(at);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (m[j]) {
            const int to = at + lanes_below(m[j]);
            if (x[8 * u + j] >= floor && to < TOP_CAP) l.e[to] = top_entry(x[8 * u + j], first + u * TOP_STEP + step(j));
            at += __popcll(m[j]);
          }
      }
    __syncthreads();
    const int more = __builtin_amdgcn_readfirstlane(*added);
    ++tile;
    if (held + more > TOP_CAP) return false;
    held += more;
    tile_done();
    return true;
  }
  // M tokens have reached a threshold that was found: later ones that only equal it are past them.
  __device__ __forceinline__ void tile_done() {
    if (limit != before) --limit;
  }

  // The list without what the threads' maxima show to be past the M-th, if longer than `few` (R = 64,
  // V = 151,936, M = 5: 20.3 us with every list trimmed, 18.1 where longer than the join takes).
  __device__ __forceinline__ void trim(TopList& l, float most, int few) {
    if (held <= few || tile == 1) return;  // (after one tile the list is at its threshold)
    const uint32_t t = top_threshold(l, fkey_desc(most), TOP_ALL, M, by);
    held = top_cut(l, held, (uint64_t)t << 32 | 0xFFFFFFFFu);
  }
};

// A tile of which too many tokens at once reach the threshold (ties, or a run of large ones): slot by slot,
// the list cut in between. load(slot, x): the thread's eight tokens of a slot.
template <int U, class F, class S>
__device__ __forceinline__ void top_slots(TopList& l, TopRun& r, int first, F load, S step) {
#pragma unroll 1
  for (int u = 0; u < U; ++u) {
    if (r.held > TOP_T) r.held = top_reduce(l, r.held, r.M, r.limit);
    const float floor = fkey_desc_inv(r.limit);
    float x[8];
    load(u, x);
    __syncthreads();
    if (threadIdx.x == 0) l.n = r.held;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (x[j] >= floor) l.e[atomicAdd(&l.n, 1)] = top_entry(x[j], first + u * TOP_STEP + step(j));
    __syncthreads();
    r.held = __builtin_amdgcn_readfirstlane(l.n);
    __syncthreads();
  }
  r.tile_done();
}

// put(place, key) for the list's first M entries; a key's place is the number of smaller ones.
template <class F>
__device__ __forceinline__ void top_order(TopList& l, int n, int M, F put) {
  uint32_t unused = 0;
  if (n > 2 * TOP_T) n = top_reduce(l, n, M, unused);
  for (int at = threadIdx.x; at < n; at += TOP_T) l.e[at] = top_key(l.e[at]);
  __syncthreads();
  for (int at = threadIdx.x; at < n; at += TOP_T) {
    const uint64_t k = l.e[at];
    int r = 0;
    for (int j = 0; j < n; ++j) r += l.e[j] < k ? 1 : 0;
    if (r < M) put(r, k);
  }
}

}  // namespace strim
