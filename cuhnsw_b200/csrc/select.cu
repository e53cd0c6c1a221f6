// The best continuations of a sequence's beams, and their states in that order.
//
//   total[b, v] = totals[b] + scores[b, v] - log sum over u of exp(scores[b, u])       (the last term if asked for)
//
// and of each sequence the `keep` largest totals over all b and v, ties to the smaller b, then the smaller v.  A total of
// -inf or NaN is never chosen.  With one beam and no normalisation these are the closest rows of an exhaustive search.
#include <float.h>

#include "common.cuh"
#include "table_common.cuh"

namespace hnsw {

namespace {

constexpr int kThreads = 256;

// A candidate of one row of scores: the order-preserving image of the score over the complement of its place, so that the
// larger key is the larger score or, of equal ones, the smaller place.  0: no candidate.
using ScoreKey = unsigned long long;
__device__ __forceinline__ ScoreKey score_key(float score, unsigned place) {
  if (!(score > -INFINITY)) return 0;
  return ((ScoreKey)f2ord(score) << 32) | (unsigned)~place;
}
__device__ __forceinline__ float key_score(ScoreKey k) { return ord2f((unsigned)(k >> 32)); }
__device__ __forceinline__ unsigned key_place(ScoreKey k) { return ~(unsigned)k; }

// The same over a sequence: totals differ by less than fp32 resolves where two beams meet, so they are compared in 64 bits.
struct TotalKey {
  unsigned long long total;  // order-preserving image of the double; 0: no candidate
  unsigned long long place;  // beam << 32 | place: the smaller one first
};
__device__ __forceinline__ unsigned long long d2ord(double x) {
  const long long u = __double_as_longlong(x + 0.0);
  return u < 0 ? ~(unsigned long long)u : (unsigned long long)u | 0x8000000000000000ull;
}
__device__ __forceinline__ double ord2d(unsigned long long o) {
  return __longlong_as_double((o & 0x8000000000000000ull) ? (long long)(o & 0x7fffffffffffffffull) : (long long)~o);
}
__device__ __forceinline__ bool above(ScoreKey a, ScoreKey b) { return a > b; }
__device__ __forceinline__ bool above(const TotalKey& a, const TotalKey& b) {
  return a.total > b.total || (a.total == b.total && a.place < b.place);
}
__device__ __forceinline__ bool none(const TotalKey& k) { return k.total == 0; }
__device__ __forceinline__ void clear(ScoreKey& k) { k = 0; }
__device__ __forceinline__ void clear(TotalKey& k) { k = {0, 0}; }

__device__ __forceinline__ ScoreKey from_lane(ScoreKey k, int lane) { return shfl64(k, lane); }
__device__ __forceinline__ TotalKey from_lane(const TotalKey& k, int lane) {
  return {shfl64(k.total, lane), shfl64(k.place, lane)};
}

// Candidates of a CTA in shared memory, in any order; `sort` puts them in descending order.
template <class Key>
struct Pool {
  Key* keys;
  int* count;
  int capacity;  // a power of two

  __device__ void push(const Key& k) { keys[atomicAdd(count, 1)] = k; }

  // All threads.  Up to a warp's worth are ranked by one warp, up to a CTA's against each other; more go through a bitonic
  // network over the smallest power of two that holds them.
  __device__ void sort() {
    __syncthreads();
    const int held = *count;
    if (held <= 32) {
      if (threadIdx.x < 32) {
        Key mine;
        clear(mine);
        if ((int)threadIdx.x < held) mine = keys[threadIdx.x];
        int rank = 0;
        for (int i = 0; i < held; ++i) rank += above(from_lane(mine, i), mine);
        __syncwarp();
        if ((int)threadIdx.x < held) keys[rank] = mine;
      }
      __syncthreads();
      return;
    }
    if (held <= kThreads) {
      Key mine;
      clear(mine);
      int rank = 0;
      if ((int)threadIdx.x < held) {
        mine = keys[threadIdx.x];
#pragma unroll 4
        for (int i = 0; i < held; ++i) rank += above(keys[i], mine);
      }
      __syncthreads();
      if ((int)threadIdx.x < held) keys[rank] = mine;
      __syncthreads();
      return;
    }
    int size = 2 * kThreads;
    while (size < held) size <<= 1;
    for (int i = held + threadIdx.x; i < size; i += kThreads) clear(keys[i]);
    for (int span = 2; span <= size; span <<= 1) {
      for (int step = span / 2; step > 0; step >>= 1) {
        __syncthreads();
        for (int i = threadIdx.x; i < size / 2; i += kThreads) {
          const int a = 2 * i - (i & (step - 1)), b = a + step;
          const bool descending = (a & span) == 0;
          const Key ka = keys[a], kb = keys[b];
          if (above(kb, ka) == descending) {
            keys[a] = kb;
            keys[b] = ka;
          }
        }
      }
    }
    __syncthreads();
  }

  // Makes room for kThreads more if there are over `most` (at most capacity - kThreads): the `keep` best stay, and `least`
  // becomes the last of them.
  __device__ void make_room(int keep, int most, Key& least) {
    __syncthreads();
    const int held = *count;
    __syncthreads();  // nobody pushes before all have read the same count
    if (held <= most) return;
    sort();
    if (threadIdx.x == 0) *count = min(*count, keep);
    __syncthreads();
    if (*count >= keep) least = keys[keep - 1];
  }
};

// ---- one piece of one row of scores ---------------------------------------------------------------------------------

// Every thread holds kEach scores.  The CTA's `keep` best: of the largest scores of twice as many groups of threads
// the `keep`-th is a bound that as many scores reach; the scores of the few threads whose largest one reaches it are looked at again,
// and what is not below goes into a pool, the pool in order.  Also the piece's largest score and its sum of
// exponentials, in fp32, which a score's place among its own beam's does not depend on: the log of a row's sum is within 3e-7 (rows of
// 1000 to 1 000 000 scores, deviations 0.01 to 30), and the same for equal rows.  (In 64 bits, by a table and a series, it is within 3e-14:
// a selection from 256 x 131 072 floats, caches cold, 69 us instead of 52.)  Bound: latency (256 x 131 072 floats in 38 us, 3.5 TB/s,
// issue slots 0.54 in use; per instruction 3.5 warps wait for loads, and 2.5 at barriers, where a CTA has no load on its way).
constexpr int kPoolScores = 4096;
constexpr int kWarps = kThreads / 32;

// Words of 16 bytes moved down by W words of 4 bytes and, if `half`, 2 bytes more: what each leaves the lane above gives, and lane 31
// the first word of the next 32 (`edges`: of 32 threads' words each).
template <int W, int Words, int Bytes>
__device__ __forceinline__ void move_words(uint4 (&word)[Words], bool half, const uint4* edges) {
  constexpr int kTaken = W + (Bytes == 2 ? 1 : 0);  // words of 4 bytes that come from above
#pragma unroll
  for (int i = 0; i < Words; ++i) {
    const uint4 edge = lane_id() == 31 ? edges[i * kWarps] : make_uint4(0, 0, 0, 0);
    const unsigned last[4] = {edge.x, edge.y, edge.z, edge.w};
    unsigned w[8] = {word[i].x, word[i].y, word[i].z, word[i].w};
#pragma unroll
    for (int k = 0; k < kTaken; ++k) {
      const unsigned above = __shfl_down_sync(FULL, w[k], 1);
      w[4 + k] = lane_id() == 31 ? last[k] : above;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = Bytes == 2 && half ? __funnelshift_r(w[k + W], w[k + W + 1], 16) : w[k + W];
    word[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <class T, int kEach>
__global__ void __launch_bounds__(kThreads, 4) piece_kernel(SelectParams p, int pieces, int piece, ScoreKey* best,
                                                         float2* norms) {
  constexpr int N = 16 / sizeof(T);
  __shared__ ScoreKey pool_keys[kPoolScores];
  __shared__ int pool_count, hot_count;
  __shared__ unsigned least_ord;
  __shared__ unsigned char hot[kThreads];  // threads whose largest score reaches the bound
  __shared__ __align__(16) float firsts[kThreads];
  __shared__ float warp_max[kWarps], warp_sum[kWarps];
  const int warp = threadIdx.x >> 5, lane = lane_id();
  next_launch_may_start();
  wait_for_launch_before();
  const long long row = blockIdx.y + (long long)blockIdx.z * 65535;
  if (row >= p.sequences * p.beams) return;
  const long long seq = row / p.beams, beam = row % p.beams;
  // Which scores a thread holds depends on their places in the row alone, not on where in memory the row begins: equal rows have
  // equal sums to the last bit, and equal totals are ties.
  constexpr int kWords = kEach / N;
  const long long begin = (long long)blockIdx.x * piece;  // of the row
  const T* scores = static_cast<const T*>(p.scores) + seq * p.seq_stride + beam * p.beam_stride + begin;
  const int skew = (int)(reinterpret_cast<uintptr_t>(scores) % 16 / sizeof(T));  // (a piece is whole words)
  const int held = (int)min((long long)piece, p.vocabulary - begin);
  if (threadIdx.x == 0) pool_count = hot_count = 0;
  float x[kEach];
  if (skew == 0) {
#pragma unroll
    for (int i = 0; i < kEach; i += N) {
      const int at = (i / N * kThreads + threadIdx.x) * N;
      if (at + N <= held) {
        const Vec<T, N> v = load_vec<T, N>(scores + at);
#pragma unroll
        for (int j = 0; j < N; ++j) x[i + j] = to_f32(v.v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[i + j] = at + j < held ? to_f32(scores[at + j]) : -INFINITY;
      }
    }
  } else {
    // Aligned words from `skew` places earlier on, then put in their places.  (Selection from 256 x 131 071 floats, caches cold: 58 us,
    // with both words of each loaded 73; 256 x 131 072: 52.)
    __shared__ uint4 edges[kWords * kWarps + 1];
    const int least = begin > 0 ? -skew : 0, last = (int)min((long long)held + N, p.vocabulary - begin);  // of the row
    auto load = [&](int at) {
      Vec<T, N> v;
      if (at >= least && at + N <= last) {
        v = load_vec<T, N>(scores + at);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v.v[j] = at + j >= least && at + j < last ? scores[at + j] : from_f32<T>(0.0f);
      }
      return *reinterpret_cast<const uint4*>(&v);
    };
    uint4 word[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) word[i] = load((int)(i * kThreads + threadIdx.x) * N - skew);
    if (threadIdx.x == 0) edges[kWords * kWarps] = load(kEach * kThreads - skew);
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) edges[i * kWarps + warp] = word[i];
    }
    __syncthreads();
    const int bytes = skew * (int)sizeof(T);
    const bool half = bytes & 2;
    switch (bytes / 4) {
      case 0: move_words<0, kWords, sizeof(T)>(word, half, edges + warp + 1); break;
      case 1: move_words<1, kWords, sizeof(T)>(word, half, edges + warp + 1); break;
      case 2: move_words<2, kWords, sizeof(T)>(word, half, edges + warp + 1); break;
      default: move_words<3, kWords, sizeof(T)>(word, half, edges + warp + 1); break;
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const Vec<T, N> v = *reinterpret_cast<const Vec<T, N>*>(&word[i]);
      const int at = (int)(i * kThreads + threadIdx.x) * N;
#pragma unroll
      for (int j = 0; j < N; ++j) x[i * N + j] = at + j < held ? to_f32(v.v[j]) : -INFINITY;
    }
  }
  float top = -INFINITY;  // (a NaN is no candidate and does not count)
#pragma unroll
  for (int i = 0; i < kEach; ++i) top = fmaxf(top, x[i]);
  // groups of `lanes` neighbouring threads, of those that have scores; their largest ones
  const int busy = min(kThreads, (held + N - 1) / N);
  int lanes = 32;
  while (lanes > 1 && kThreads / lanes < 2 * p.keep) lanes >>= 1;
  const int groups = max(0, (busy + lanes - 1) / lanes);
  float of_group = top, of_warp = top;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    of_warp = fmaxf(of_warp, __shfl_xor_sync(FULL, of_warp, off));
    if (off < lanes) of_group = of_warp;
  }
  if ((threadIdx.x & (lanes - 1)) == 0) firsts[threadIdx.x / lanes] = of_group;
  if (lane == 0) warp_max[warp] = of_warp;
  if (threadIdx.x == 0) least_ord = 0xffffffffu;
  __syncthreads();
  // the smallest of those that fewer than `keep` others exceed
  if ((int)threadIdx.x < groups) {
    const float mine = firsts[threadIdx.x];
    int larger = 0;
#pragma unroll 8
    for (int i = 0; i < groups; ++i) larger += firsts[i] > mine;
    if (larger < p.keep) atomicMin(&least_ord, f2ord(mine));
  }
  float most = -FLT_MAX;  // (of a row of -inf the exponentials are zeros)
#pragma unroll
  for (int w = 0; w < kWarps; ++w) most = fmaxf(most, warp_max[w]);
  if (p.log_softmax) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += exp2_of((x[i] - most) * 1.44269504f);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(FULL, sum, off);
    if (lane == 0) warp_sum[warp] = sum;
  }
  __syncthreads();
  // -inf is no candidate: it is less than the lowest number.  (With fewer groups than results there is no bound.)
  const float bound = groups < p.keep ? -FLT_MAX : fmaxf(ord2f(least_ord), -FLT_MAX);
  if (top >= bound) hot[atomicAdd(&hot_count, 1)] = (unsigned char)threadIdx.x;
  __syncthreads();
  const int slots = hot_count * kEach;
  Pool<ScoreKey> pool{pool_keys, &pool_count, kPoolScores};
  ScoreKey from = 0;
  for (int slot = threadIdx.x; slot - (int)threadIdx.x < slots; slot += kThreads) {
    if (slots > kPoolScores) pool.make_room(p.keep, kPoolScores - kThreads, from);
    if (slot >= slots) continue;
    const int i = slot % kEach, at = (i / N * kThreads + hot[slot / kEach]) * N + i % N;
    const float xi = at < held ? to_f32(scores[at]) : -INFINITY;
    if (xi >= bound) {
      const ScoreKey k = score_key(xi, (unsigned)(begin + at));
      if (k >= from) pool.push(k);
    }
  }
  pool.sort();
  if (p.log_softmax && threadIdx.x == 0) {
    float all = warp_sum[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) all += warp_sum[w];
    norms[row * pieces + blockIdx.x] = make_float2(most, all);
  }
  ScoreKey* to = best + (row * pieces + blockIdx.x) * p.keep;
  const int kept = min(pool_count, p.keep);
  for (int i = threadIdx.x; i < p.keep; i += kThreads) to[i] = i < kept ? pool_keys[i] : 0;
}

// ---- a sequence -----------------------------------------------------------------------------------------------------

constexpr int kPoolTotals = 2048;

__device__ __forceinline__ float score_at(const SelectParams& p, long long at) {
  if (p.type == kF32) return static_cast<const float*>(p.scores)[at];
  if (p.type == kF16) return to_f32(static_cast<const __half*>(p.scores)[at]);
  return to_f32(static_cast<const __nv_bfloat16*>(p.scores)[at]);
}

// Whether different scores, raised by `offset`, may round to the same `total`.  They are no further apart than the doubles beside the
// total, 2^-52 of it, and no closer than 2^-24 of the larger one: that is at most 2^-28 of the total.  (The rest is room for the
// roundings of the difference.  Infinities and 0 beside an offset count as such.)
__device__ __forceinline__ bool merged(double offset, double total) {
  return offset != 0.0 && !(fabs(total - offset) * 0x1p27 > fabs(total));
}

// One CTA per sequence.  The lists of the pieces are in order: of their first totals the `keep`-th is a bound that as many
// candidates reach, and from there on there are few.  Bound: latency, a chain of some ten steps.  (8 sequences of 4 beams over
// 32 000 ids, 64 lists: 25 us for a whole step of a beam search, 42 if up to 256 candidates are put in order without a bound.)
__global__ void __launch_bounds__(kThreads) sequence_kernel(SelectParams p, int pieces, int piece, const ScoreKey* best,
                                                            const float2* norms) {
  extern __shared__ __align__(16) unsigned char smem[];
  TotalKey* pool_keys = reinterpret_cast<TotalKey*>(smem);
  double* offsets = reinterpret_cast<double*>(pool_keys + kPoolTotals);  // what a beam's scores are raised by
  __shared__ int pool_count;
  __shared__ unsigned long long least_total;
  const int lane = lane_id(), warp = threadIdx.x >> 5;
  const long long seq = blockIdx.x;
  const int beams = (int)p.beams;
  const long long lists = (long long)beams * pieces, total = lists * p.keep;
  const ScoreKey* mine = best + seq * total;
  next_launch_may_start();
  if (threadIdx.x == 0) pool_count = 0;
  wait_for_launch_before();
  const ScoreKey first = (long long)threadIdx.x < lists ? mine[threadIdx.x * p.keep] : 0;  // on its way meanwhile
  for (int b = warp; b < beams; b += kWarps) {
    double offset = p.totals ? (double)p.totals[seq * beams + b] : 0.0;
    if (p.log_softmax) {
      const float2* of_row = norms + (seq * beams + b) * pieces;
      const float2 norm = lane < pieces ? of_row[lane] : make_float2(-FLT_MAX, 0.0f);
      float most = norm.x;
      for (int i = lane + 32; i < pieces; i += 32) most = fmaxf(most, of_row[i].x);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(FULL, most, off));
      double sum = norm.y * exp((double)norm.x - (double)most);
      for (int i = lane + 32; i < pieces; i += 32) sum += of_row[i].y * exp((double)of_row[i].x - (double)most);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(FULL, sum, off);
      offset -= (double)most + log(sum);
    }
    if (lane == 0) offsets[b] = offset;
  }
  __syncthreads();
  auto total_key = [&](long long list, ScoreKey k) {
    TotalKey key = {0, 0};
    if (k == 0) return key;
    const unsigned beam = (unsigned)list / (unsigned)pieces;
    const double value = offsets[beam] + (double)key_score(k);
    if (value > -INFINITY) key = {d2ord(value), (unsigned long long)beam << 32 | key_place(k)};
    return key;
  };
  Pool<TotalKey> pool{pool_keys, &pool_count, kPoolTotals};
  TotalKey least = {0, 0};
  if (total > 32) {
    // every thread one of the lists' first totals (the best of several lists', of more lists than threads), the `keep`-th of
    // them all: as many candidates reach it
    const long long heads = min((long long)kThreads, total);
    unsigned long long* totals = reinterpret_cast<unsigned long long*>(pool_keys);
    unsigned long long top = 0;
    if (lists >= kThreads) {
      for (long long list = threadIdx.x; list < lists; list += kThreads)
        top = max(top, total_key(list, list < kThreads ? first : mine[list * p.keep]).total);
    } else {
      const unsigned list = threadIdx.x % (unsigned)lists, rank = threadIdx.x / (unsigned)lists;
      if (rank < p.keep) top = total_key(list, rank == 0 ? first : mine[(long long)list * p.keep + rank]).total;
    }
    totals[threadIdx.x] = top;
    if (threadIdx.x == 0) least_total = ~0ull;
    __syncthreads();
    int larger = 0;
#pragma unroll 8
    for (int i = 0; i < kThreads; ++i) larger += totals[i] > top;
    if (larger < p.keep) atomicMin(&least_total, top);
    __syncthreads();
    // (places of the largest order: all of this total are above it)
    if (heads >= p.keep) least = {least_total, ~0ull};
    __syncthreads();
  }
  // All lists' totals of a rank after those of the one before, until none of a whole rank reaches the bound: the lists are in
  // order.
  const bool narrow = total < (1ll << 32);
  auto candidate = [&](long long i) { return i < total ? mine[(narrow ? (unsigned)i % (unsigned)lists : i % lists) * p.keep +
                                                              (narrow ? (unsigned)i / (unsigned)lists : i / lists)] : 0; };
  ScoreKey next = candidate(threadIdx.x);
  long long below = 0;
  for (long long begin = 0; begin < total; begin += kThreads) {
    if (begin > 0) pool.make_room(p.keep, 2 * p.keep + 32, least);  // (the sooner the bound rises the less there is to sort)
    const long long i = begin + threadIdx.x;
    const ScoreKey k = next;
    next = candidate(i + kThreads);
    const TotalKey key = total_key(narrow ? (unsigned)i % (unsigned)lists : i % lists, k);
    const bool reaches = !none(key) && !above(least, key);
    if (reaches) pool.push(key);
    below = __syncthreads_or(reaches) ? 0 : below + kThreads;
    if (below >= lists) break;
  }
  pool.sort();
  const int found = min(pool_count, p.keep);
  // A list has its piece's best scores.  What it lacks can only matter in totals equal to the last result's, of a beam whose
  // offset gives different scores the same total: then the results of that total are looked for again, in the order of the places.
  // (Found fewer than `keep`: the lists lack nothing.)
  const bool one = (int)threadIdx.x < found;
  const TotalKey own = one ? pool_keys[threadIdx.x] : TotalKey{0, 0};
  const unsigned long long border = pool_keys[max(found - 1, 0)].total;
  if (__syncthreads_or(one && found == p.keep && own.total == border && merged(offsets[own.place >> 32], ord2d(border)))) {
    __shared__ unsigned masks[2][kWarps];
    int taken = __syncthreads_count(one && own.total > border);  // of the results
    for (long long base = 0; base < lists && taken < found; base += kThreads) {
      // pieces that have such a total: their lists begin at or above it and do not end above it
      const long long mine_list = base + threadIdx.x;
      const bool has = mine_list < lists && total_key(mine_list, mine[mine_list * p.keep]).total >= border &&
                       total_key(mine_list, mine[mine_list * p.keep + p.keep - 1]).total <= border;
      const unsigned having = __ballot_sync(FULL, has);
      if (lane == 0) masks[0][warp] = having;
      __syncthreads();
      for (int w = 0; w < kWarps; ++w) {
        for (unsigned left = masks[0][w]; left && taken < found; left &= left - 1) {
          const unsigned list = (unsigned)base + 32 * w + __ffs(left) - 1, beam = list / (unsigned)pieces;
          const long long begin = (long long)(list % (unsigned)pieces) * piece, end = min(begin + piece, p.vocabulary);
          const long long row = seq * p.seq_stride + beam * p.beam_stride;
          for (long long at = begin; at < end && taken < found; at += kThreads) {
            const long long v = at + threadIdx.x;
            const float score = v < end ? score_at(p, row + v) : -INFINITY;
            const bool same = score > -INFINITY && d2ord(offsets[beam] + (double)score) == border;
            const unsigned all = __ballot_sync(FULL, same);
            if (lane == 0) masks[1][warp] = all;
            __syncthreads();
            int before = taken + __popc(all & ((1u << lane) - 1));
            for (int other = 0; other < kWarps; ++other) {
              before += other < warp ? __popc(masks[1][other]) : 0;
              taken += __popc(masks[1][other]);
            }
            if (same && before < found) pool_keys[before] = {border, (unsigned long long)beam << 32 | (unsigned)v};
            __syncthreads();
          }
        }
      }
      __syncthreads();
    }
  }
  for (int i = threadIdx.x; i < p.keep; i += kThreads) {
    const TotalKey k = pool_keys[i];
    const long long at = seq * p.keep + i;
    p.out_totals[at] = p.sign * (i < found ? (float)ord2d(k.total) : -INFINITY);
    if (p.out_beams) p.out_beams[at] = i < found ? (int)(k.place >> 32) : -1;
    p.out_ids[at] = i < found ? (int)(unsigned)k.place : -1;
  }
  if (p.out_found && threadIdx.x == 0) p.out_found[seq] = found;
}

struct SelectPlan {
  int each;           // scores per thread at most
  int piece;          // scores: whole words
  long long pieces;
};
SelectPlan select_plan(long long rows, long long vocabulary) {
  SelectPlan s;
  // Pieces of up to 8192 scores where that still gives every SM four of them, all of about the same length.  (A step of a beam
  // search, 32 x 8 beams of 131 072 ids: 89 us, with pieces of 2048 127; 1 x 4 of 32 000: 27 us with 2048, 33 with 8192.)
  s.each = 32;
  while (s.each > 8 && rows * ((vocabulary + kThreads * s.each - 1) / (kThreads * s.each)) < 4 * kSMs) s.each /= 2;
  s.pieces = (vocabulary + kThreads * s.each - 1) / (kThreads * s.each);
  s.piece = (int)(((vocabulary + s.pieces - 1) / s.pieces + 7) / 8 * 8);
  return s;
}

template <class T>
cudaError_t pieces_t(const SelectParams& p, const SelectPlan& plan, ScoreKey* best, float2* norms, cudaStream_t stream) {
  const long long rows = p.sequences * p.beams;
  const dim3 grid((unsigned)plan.pieces, (unsigned)(rows < 65535 ? rows : 65535), (unsigned)((rows + 65534) / 65535));
  if (plan.each == 32)
    return launch_early(piece_kernel<T, 32>, grid, kThreads, 0, stream, p, (int)plan.pieces, plan.piece, best, norms);
  if (plan.each == 16)
    return launch_early(piece_kernel<T, 16>, grid, kThreads, 0, stream, p, (int)plan.pieces, plan.piece, best, norms);
  return launch_early(piece_kernel<T, 8>, grid, kThreads, 0, stream, p, (int)plan.pieces, plan.piece, best, norms);
}

// ---- states ---------------------------------------------------------------------------------------------------------

struct ReorderParams {
  ReorderState state[kMaxStates];
  int word[kMaxStates];
  const int* beams_of;
  long long sequences;
  long long beams;
  long long keep;
};

template <class W>
__device__ __forceinline__ void copy_row(const ReorderState& s, const char* from, char* to) {
  const long long words = s.bytes / (long long)sizeof(W), all = words * s.segments;
  const long long step = (long long)gridDim.x * kThreads;
  W* dst = reinterpret_cast<W*>(to);
  for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < all; i += step) {
    W w{};
    if (from) {
      const long long segment = s.segments == 1 ? 0 : i / words, at = s.segments == 1 ? i : i % words;
      w = __ldcs(reinterpret_cast<const W*>(from + segment * s.segment_stride) + at);
    }
    __stcs(dst + i, w);
  }
}

// Grid: pieces of a row x rows x states.  Bound: HBM bytes (134 MB there and back in 42 us, from the L2 cache in part).
__global__ void __launch_bounds__(kThreads) reorder_kernel(const __grid_constant__ ReorderParams p) {
  next_launch_may_start();
  wait_for_launch_before();
  const ReorderState& s = p.state[blockIdx.z];
  const long long rows = p.sequences * p.keep;
  for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
    const long long seq = row / p.keep;
    const int beam = p.beams_of[row];
    const char* from = beam < 0 || beam >= p.beams
                         ? nullptr
                         : static_cast<const char*>(s.src) + seq * s.seq_stride + beam * s.beam_stride;
    char* to = static_cast<char*>(s.dst) + row * s.segments * s.bytes;
    switch (p.word[blockIdx.z]) {
      case 16: copy_row<uint4>(s, from, to); break;
      case 8: copy_row<uint2>(s, from, to); break;
      case 4: copy_row<unsigned>(s, from, to); break;
      case 2: copy_row<unsigned short>(s, from, to); break;
      default: copy_row<unsigned char>(s, from, to); break;
    }
  }
}

size_t best_bytes(long long rows, long long pieces, int keep) {
  return ((size_t)rows * pieces * keep * sizeof(ScoreKey) + 255) / 256 * 256;
}

}  // namespace

size_t select_workspace(long long sequences, long long beams, long long vocabulary, int keep) {
  if (sequences <= 0 || beams <= 0 || vocabulary <= 0) return 0;
  const long long rows = sequences * beams, pieces = select_plan(rows, vocabulary).pieces;
  return best_bytes(rows, pieces, keep) + (size_t)rows * pieces * sizeof(float2);
}

cudaError_t launch_select(const SelectParams& p, cudaStream_t stream) {
  if (p.sequences <= 0) return cudaSuccess;
  const long long rows = p.sequences * p.beams;
  const SelectPlan plan = select_plan(rows, p.vocabulary);
  const size_t smem = kPoolTotals * sizeof(TotalKey) + (size_t)p.beams * sizeof(double);
  if (p.sequences > 0x7fffffffll || plan.pieces > 0x7fffffffll || rows > 65535ll * 65535 || smem > 200 * 1024)
    return cudaErrorInvalidValue;
  ScoreKey* best = static_cast<ScoreKey*>(p.workspace);
  float2* norms = reinterpret_cast<float2*>(static_cast<char*>(p.workspace) + best_bytes(rows, plan.pieces, p.keep));
  cudaError_t e = p.type == kF32   ? pieces_t<float>(p, plan, best, norms, stream)
                  : p.type == kF16 ? pieces_t<__half>(p, plan, best, norms, stream)
                                   : pieces_t<__nv_bfloat16>(p, plan, best, norms, stream);
  if (e != cudaSuccess) return e;
  e = allow_smem<sequence_kernel>();
  if (e != cudaSuccess) return e;
  return launch_early(sequence_kernel, dim3((unsigned)p.sequences), kThreads, smem, stream, p, (int)plan.pieces, plan.piece, best,
                      norms);
}

cudaError_t launch_reorder(const ReorderState* states, int count, const int* beams_of, long long sequences,
                           long long beams, long long keep, cudaStream_t stream) {
  const long long rows = sequences * keep;
  if (rows <= 0 || count <= 0) return cudaSuccess;
  ReorderParams p;
  long long most = 0;
  for (int i = 0; i < count; ++i) {
    const ReorderState& s = states[i];
    p.state[i] = s;
    p.word[i] = word_bytes(reinterpret_cast<uintptr_t>(s.src) | reinterpret_cast<uintptr_t>(s.dst) |
                           (unsigned long long)s.seq_stride | (unsigned long long)s.beam_stride |
                           (unsigned long long)(s.segments > 1 ? s.segment_stride : 0) | (unsigned long long)s.bytes);
    const long long words = s.segments * (s.bytes / p.word[i]);
    most = words > most ? words : most;
  }
  if (most == 0) return cudaSuccess;
  p.beams_of = beams_of;
  p.sequences = sequences;
  p.beams = beams;
  p.keep = keep;
  const long long pieces = (most + 4 * kThreads - 1) / (4 * kThreads);
  const dim3 grid((unsigned)(pieces < 4096 ? pieces : 4096), (unsigned)(rows < 65535 ? rows : 65535), (unsigned)count);
  return launch_early(reorder_kernel, grid, kThreads, 0, stream, p);
}

}  // namespace hnsw
