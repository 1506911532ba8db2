// top.hpp — the first M tokens of a row in token order (logit descending, then id), M <= TOP_MAX, by one
// workgroup of TOP_T threads that meets the row a tile at a time.
//
// Each thread keeps the largest logit it has met. The M-th largest of the threads' maxima is no larger
// than the M-th largest logit met so far, and hardly smaller: with 256 threads and M = 64 about 74
// logits reach it. So tokens that reach this threshold are appended to a list in LDS, one of its own for
// each wave (no atomics, and the waves meet only where the threshold is raised: after tiles 1, 2, 4, 8,
// ...; between two of them about M tokens are appended), and at the end the lists are cut at the last
// threshold, joined and ordered. Ids ascend from tile to tile: once M tokens have reached a threshold, a
// later one that only equals it is past the M-th.
#pragma once

#include "common.hpp"

namespace strim {

constexpr int TOP_T = 256;
constexpr int TOP_MAX = STRIM_SCORE_MAX_LIST;
constexpr int TOP_STEP = 2048;             // tokens a workgroup appends at most between two looks at a list's length
constexpr int TOP_CAP = TOP_STEP + TOP_T;  // list: what was there when it was last cut, and a step
constexpr int TOP_WAVES = TOP_T / WAVE;
constexpr int TOP_ROOM = TOP_CAP / TOP_WAVES;  // a wave's list
static_assert(TOP_MAX <= TOP_T && TOP_MAX + WAVE <= TOP_ROOM, "a list that was cut leaves room for a step");
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
  uint64_t e[TOP_CAP];   // entries, in no order: TOP_ROOM a wave, or one list
  uint32_t best[TOP_T];  // fkey_desc of the threads' maxima
  uint32_t limit;
  int n;
  int part[2][TOP_WAVES];
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

// A wave's view of its list while the row goes by.
struct TopRun {
  uint64_t* e;            // the wave's list
  int held, tile;         // its entries; tiles met
  uint32_t limit, own;    // tokens whose fkey_desc is at most both are appended: the workgroup's limit, the wave's
  int M, by;
  uint32_t before, mine;  // the limits before this tile

  __device__ __forceinline__ void init(TopList& l, int m) {
    e = l.e + wave_id() * TOP_ROOM;
    by = blockIdx.x % TOP_WAVES;
    held = tile = 0;
    limit = own = TOP_ALL;
    M = m;
  }

  // A tile of U slots of TOP_STEP tokens, eight a thread: x[8 u ..] are the thread's of slot u, with ids
  // first + u TOP_STEP + step(j); mv[u] is their maximum, `most` the largest that the thread has met. False where
  // the wave would append more than its list holds: the tile is then given to top_slots.
  template <int U, class S>
  __device__ __forceinline__ bool add(TopList& l, const float (&x)[8 * U], const float (&mv)[U], float most, int first,
                                      S step) {
    before = limit;
    mine = own;
    if (((tile + 1) & tile) == 0) limit = top_threshold(l, fkey_desc(most), limit, M, by);
    const float floor = least();
    const int was = held;
    ++tile;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (__ballot(mv[u] >= floor)) {
        uint64_t m[8];
        int n = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          m[j] = __ballot(x[8 * u + j] >= floor);
          n += __popcll(m[j]);
        }
        if (held + n > TOP_ROOM) {
          held = was;
          return false;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (m[j]) {
            if (x[8 * u + j] >= floor)
              e[held + lanes_below(m[j])] = top_entry(x[8 * u + j], first + u * TOP_STEP + step(j));
            held += __popcll(m[j]);
          }
      }
    tile_done();
    return true;
  }
  __device__ __forceinline__ float least() const { return fkey_desc_inv(min(limit, own)); }
  // M tokens have reached a limit that was found in this tile: later ones that only equal it are past them.
  __device__ __forceinline__ void tile_done() {
    if (limit != before) --limit;
    if (own != mine) --own;
  }

  // The wave's list cut to its first M entries; its limit is lowered to the last one's logit (tokens of the
  // same tile that equal it may still come before it). held > M.
  __device__ __forceinline__ void cut() {
    constexpr int Q = TOP_ROOM / WAVE;
    const int lane = threadIdx.x & (WAVE - 1);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint64_t v[Q];
    uint32_t k[Q];
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      v[i] = i * WAVE + lane < held ? e[i * WAVE + lane] : TOP_NONE;
      k[i] = i * WAVE + lane < held ? fkey_desc(__uint_as_float((uint32_t)(v[i] >> 32))) : ~0u;
    }
    auto reach = [&](uint32_t t) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < Q; ++i) n += __popcll(__ballot(k[i] <= t));
      return n;
    };
    uint32_t lo = ~0u, hi = 0;
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      lo = min(lo, k[i]);
      hi = max(hi, i * WAVE + lane < held ? k[i] : 0u);
    }
    // (the reductions are of signed numbers) reach(hi) >= M > reach(lo)
    lo = ((uint32_t)wave_min_i((int)(lo ^ 0x80000000u)) ^ 0x80000000u) - 1u;
    hi = (uint32_t)wave_max_i((int)(hi ^ 0x80000000u)) ^ 0x80000000u;
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (reach(mid) >= M) hi = mid;
      else lo = mid;
    }
    // of those that equal the M-th the lower ids
    const int extra = reach(hi) - M;
    uint32_t id = ~0u;
    if (extra > 0) {
      const int all = M - reach(hi - 1);          // how many of them stay
      uint32_t a = 0, b = STRIM_SCORE_MAX_VOCAB;  // ids below a: fewer than `all`; below b: as many at least
      while (b - a > 1) {
        const uint32_t mid = a + (b - a) / 2;
        int n = 0;
#pragma unroll
        for (int i = 0; i < Q; ++i) n += __popcll(__ballot(k[i] == hi && (uint32_t)v[i] < mid));
        if (n >= all) b = mid;
        else a = mid;
      }
      id = b;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    int at = 0;
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const bool stays = k[i] < hi || (k[i] == hi && (uint32_t)v[i] < id);
      const uint64_t b = __ballot(stays);
      if (stays) e[at + lanes_below(b)] = v[i];
      at += __popcll(b);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    held = at;
    own = min(own, hi);
  }

  // The wave's length for the others, who see it after a barrier of the caller's; then where its entries begin
  // among the `all` of the workgroup.
  __device__ __forceinline__ void leave(TopList& l) const {
    if ((threadIdx.x & (WAVE - 1)) == 0) l.part[0][wave_id()] = held;
  }
  __device__ __forceinline__ int place(const TopList& l, int& all) const {
    int at = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < TOP_WAVES; ++i) {
      if (i < wave_id()) at += l.part[0][i];
      sum += l.part[0][i];
    }
    all = __builtin_amdgcn_readfirstlane(sum);
    return __builtin_amdgcn_readfirstlane(at);
  }

  // The waves' lists as one from l.e on, without what the threads' maxima show to be past the M-th. All threads;
  // returns its length.
  __device__ __forceinline__ int gather(TopList& l, float most) {
    constexpr int Q = TOP_ROOM / WAVE;
    const int lane = threadIdx.x & (WAVE - 1), wave = wave_id();
    uint32_t last = TOP_ALL;
    if (tile > 1) last = top_threshold(l, fkey_desc(most), TOP_ALL, M, by);  // (one tile's lists are at theirs)
    uint64_t v[Q], b[Q];
    int n = 0;
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const bool in = i * WAVE + lane < held;
      v[i] = in ? e[i * WAVE + lane] : TOP_NONE;
      b[i] = __ballot(in && fkey_desc(__uint_as_float((uint32_t)(v[i] >> 32))) <= last);
      n += __popcll(b[i]);
    }
    if (lane == 0) l.part[1][wave] = n;
    __syncthreads();
    int at = 0, all = 0;
#pragma unroll
    for (int i = 0; i < TOP_WAVES; ++i) {
      if (i < wave) at += l.part[1][i];
      all += l.part[1][i];
    }
    at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      if ((b[i] >> lane) & 1u) l.e[at + lanes_below(b[i])] = v[i];
      at += __popcll(b[i]);
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(all);
  }
};

// A tile of which too many of a wave's tokens at once reach the threshold (ties, or a run of large ones): a
// token of each lane after another, the list cut in between. load(slot, x): the thread's eight tokens of a slot.
template <int U, class F, class S>
__device__ __forceinline__ void top_slots(TopRun& r, int first, F load, S step) {
#pragma unroll 1
  for (int u = 0; u < U; ++u) {
    float x[8];
    load(u, x);
#pragma unroll 1
    for (int j = 0; j < 8; ++j) {
      float f = x[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) f = j == i ? x[i] : f;
      uint64_t m = __ballot(f >= r.least());
      if (r.held + __popcll(m) > TOP_ROOM) {
        r.cut();
        m = __ballot(f >= r.least());
      }
      if ((m >> (threadIdx.x & (WAVE - 1))) & 1u) r.e[r.held + lanes_below(m)] = top_entry(f, first + u * TOP_STEP + step(j));
      r.held += __popcll(m);
    }
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
