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
  unsigned place;
  unsigned beam;
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
  if (a.total != b.total) return a.total > b.total;
  if (a.beam != b.beam) return a.beam < b.beam;
  return a.place < b.place;
}
__device__ __forceinline__ bool none(const TotalKey& k) { return k.total == 0; }
__device__ __forceinline__ void clear(ScoreKey& k) { k = 0; }
__device__ __forceinline__ void clear(TotalKey& k) { k = {0, 0, 0}; }

__device__ __forceinline__ ScoreKey from_lane(ScoreKey k, int lane) { return shfl64(k, lane); }
__device__ __forceinline__ TotalKey from_lane(const TotalKey& k, int lane) {
  return {shfl64(k.total, lane), __shfl_sync(FULL, k.place, lane), __shfl_sync(FULL, k.beam, lane)};
}

// Candidates of a CTA in shared memory, in any order; `sort` puts them in descending order.
template <class Key>
struct Pool {
  Key* keys;
  int* count;
  int capacity;  // a power of two

  __device__ void push(const Key& k) { keys[atomicAdd(count, 1)] = k; }

  // All threads.  Up to a warp's worth are ranked by one warp; more go through a bitonic network over the smallest power of two
  // that holds them.
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
    int size = 64;
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

  // Makes room for kThreads more if there is none: the `keep` best stay, and `least` becomes the last of them.
  __device__ void make_room(int keep, Key& least) {
    __syncthreads();
    const int held = *count;
    __syncthreads();  // nobody pushes before all have read the same count
    if (held + kThreads <= capacity) return;
    sort();
    if (threadIdx.x == 0) *count = min(*count, keep);
    __syncthreads();
    if (*count >= keep) least = keys[keep - 1];
  }
};

// ---- one piece of one row of scores ---------------------------------------------------------------------------------

// Every thread holds kEach scores.  The CTA's `keep` best: a bound that at least `keep` of them reach (groups of threads
// are at least that many, and the smallest of the groups' largest scores is reached once in each), everything from there on
// into a pool, the pool in order.  Also the piece's largest score and its sum of exponentials.  Bound: HBM bytes, and the
// instructions for every score: its part in the maximum, in the sum, and one comparison.
constexpr int kPoolScores = 2048;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <class T, int N, int kEach>
__global__ void __launch_bounds__(kThreads) piece_kernel(SelectParams p, int pieces, ScoreKey* best, float2* norms) {
  __shared__ ScoreKey pool_keys[kPoolScores];
  __shared__ int pool_count;
  __shared__ float firsts[kThreads];
  __shared__ float warp_max[kWarps], warp_sum[kWarps];
  const int warp = threadIdx.x >> 5, lane = lane_id();
  const long long row = blockIdx.y + (long long)blockIdx.z * 65535;
  if (row >= p.sequences * p.beams) return;
  const long long seq = row / p.beams, beam = row % p.beams;
  const T* scores = static_cast<const T*>(p.scores) + seq * p.seq_stride + beam * p.beam_stride;
  const int vocabulary = (int)p.vocabulary;
  const unsigned begin = blockIdx.x * (unsigned)(kThreads * kEach);  // (below 2^31, and so is the vocabulary)
  auto place = [&](int i) { return begin + (unsigned)((i / N * kThreads + threadIdx.x) * N + i % N); };
  if (threadIdx.x == 0) pool_count = 0;
  float x[kEach];
#pragma unroll
  for (int i = 0; i < kEach; i += N) {
    const unsigned at = place(i);
    if (at + N <= (unsigned)vocabulary) {
      const Vec<T, N> v = load_stream<T, N>(scores + at);
#pragma unroll
      for (int j = 0; j < N; ++j) x[i + j] = to_f32(v.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) x[i + j] = at + j < (unsigned)vocabulary ? to_f32(scores[at + j]) : -INFINITY;
    }
  }
  float top = x[0];
#pragma unroll
  for (int i = 1; i < kEach; ++i) top = fmaxf(top, x[i]);
  // groups of `lanes` threads, at least `keep` of them; their largest scores
  int lanes = kThreads;
  while (lanes > 1 && kThreads / lanes < p.keep) lanes >>= 1;
  float of_group = top, of_warp = top;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    of_warp = fmaxf(of_warp, __shfl_xor_sync(FULL, of_warp, off));
    if (off < lanes) of_group = of_warp;
  }
  firsts[threadIdx.x] = of_group;
  if (lane == 0) warp_max[warp] = of_warp;
  __syncthreads();
  float most = -FLT_MAX, least = INFINITY;  // (of a row of -inf the exponentials are zeros)
  if (lanes <= 32) {
    for (int i = lane * lanes; i < kThreads; i += 32 * lanes) least = fminf(least, firsts[i]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) least = fminf(least, __shfl_xor_sync(FULL, least, off));
  } else {
    for (int w = 0; w < kWarps; w += lanes / 32) {
      float of_warps = warp_max[w];
      for (int v = 1; v < lanes / 32; ++v) of_warps = fmaxf(of_warps, warp_max[w + v]);
      least = fminf(least, of_warps);
    }
  }
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
  // -inf and NaN are no candidates: neither is at least the lowest number.  (A group without scores has no largest one.)
  const float bound = fmaxf(least, -FLT_MAX);
  int passing = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) passing += x[i] >= bound;
  Pool<ScoreKey> pool{pool_keys, &pool_count, kPoolScores};
  if (__syncthreads_or(passing > kPoolScores / kThreads) == 0) {
    if (passing > 0) {
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (x[i] >= bound) pool.push(score_key(x[i], place(i)));
    }
  } else {
    // so many that they may not fit: a score of each thread at a time
    ScoreKey from = 0;
#pragma unroll 1
    for (int i = 0; i < kEach; ++i) {
      pool.make_room(p.keep, from);
      float xi = x[0];
#pragma unroll
      for (int j = 1; j < kEach; ++j) xi = j == i ? x[j] : xi;
      const ScoreKey k = score_key(xi, place(i));
      if (xi >= bound && k >= from) pool.push(k);
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
  const int held = min(pool_count, p.keep);
  for (int i = threadIdx.x; i < p.keep; i += kThreads) to[i] = i < held ? pool_keys[i] : 0;
}

// ---- a sequence -----------------------------------------------------------------------------------------------------

constexpr int kPoolTotals = 2048;

// One CTA per sequence.  The lists of the pieces are in order: of their first totals the `keep`-th is a bound that as many
// candidates reach, and from there on there are few.
__global__ void __launch_bounds__(kThreads) sequence_kernel(SelectParams p, int pieces, const ScoreKey* best,
                                                            const float2* norms) {
  extern __shared__ __align__(16) unsigned char smem[];
  TotalKey* pool_keys = reinterpret_cast<TotalKey*>(smem);
  double* offsets = reinterpret_cast<double*>(pool_keys + kPoolTotals);  // what a beam's scores are raised by
  __shared__ int pool_count;
  const int lane = lane_id(), warp = threadIdx.x >> 5;
  const long long seq = blockIdx.x;
  const int beams = (int)p.beams;
  const long long lists = (long long)beams * pieces, total = lists * p.keep;
  const ScoreKey* mine = best + seq * total;
  if (threadIdx.x == 0) pool_count = 0;
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
    TotalKey key = {0, 0, 0};
    if (k == 0) return key;
    const unsigned beam = (unsigned)list / (unsigned)pieces;
    const double value = offsets[beam] + (double)key_score(k);
    if (value > -INFINITY) key = {d2ord(value), key_place(k), beam};
    return key;
  };
  Pool<TotalKey> pool{pool_keys, &pool_count, kPoolTotals};
  TotalKey least = {0, 0, 0};
  if (lists >= p.keep && total > kThreads) {
    // the best first total of each thread's lists, the `keep`-th of them all
    TotalKey top = total_key(threadIdx.x, first);
    for (long long list = threadIdx.x + kThreads; list < lists; list += kThreads) {
      const TotalKey key = total_key(list, mine[list * p.keep]);
      if (above(key, top)) top = key;
    }
    pool_keys[threadIdx.x] = top;
    __syncthreads();
    const int held = (int)min((long long)kThreads, lists);
    int rank = 0;
    if (!none(top))
      for (int i = 0; i < held; ++i) rank += above(pool_keys[i], top);
    __syncthreads();
    if (!none(top) && rank == p.keep - 1) pool_keys[0] = top;
    const bool there = __syncthreads_or(!none(top) && rank == p.keep - 1);
    if (there) least = pool_keys[0];
    __syncthreads();
  }
  // list by list of the same rank: the best ones first
  for (long long begin = 0; begin < total; begin += kThreads) {
    pool.make_room(p.keep, least);
    const long long i = begin + threadIdx.x;
    if (i < total) {
      const unsigned long long list = total < (1ll << 32) ? (unsigned)i % (unsigned)lists : i % lists;
      const unsigned long long rank = total < (1ll << 32) ? (unsigned)i / (unsigned)lists : i / lists;
      const TotalKey key = total_key(list, mine[list * p.keep + rank]);
      if (!none(key) && !above(least, key)) pool.push(key);
    }
  }
  pool.sort();
  const int found = min(pool_count, p.keep);
  for (int i = threadIdx.x; i < p.keep; i += kThreads) {
    const TotalKey k = pool_keys[i];
    const long long at = seq * p.keep + i;
    p.out_totals[at] = p.sign * (i < found ? (float)ord2d(k.total) : -INFINITY);
    if (p.out_beams) p.out_beams[at] = i < found ? (int)k.beam : -1;
    p.out_ids[at] = i < found ? (int)k.place : -1;
  }
  if (p.out_found && threadIdx.x == 0) p.out_found[seq] = found;
}

struct SelectPlan {
  int each;
  long long pieces;
};
SelectPlan select_plan(long long rows, long long vocabulary) {
  SelectPlan s;
  // pieces of 8192 scores where that still gives every SM four of them
  s.each = 32;
  while (s.each > 8 && rows * ((vocabulary + kThreads * s.each - 1) / (kThreads * s.each)) < 4 * kSMs) s.each /= 2;
  s.pieces = (vocabulary + kThreads * s.each - 1) / (kThreads * s.each);
  return s;
}

template <class T, int N>
cudaError_t pieces_t(const SelectParams& p, const SelectPlan& plan, ScoreKey* best, float2* norms, cudaStream_t stream) {
  const long long rows = p.sequences * p.beams;
  const dim3 grid((unsigned)plan.pieces, (unsigned)(rows < 65535 ? rows : 65535), (unsigned)((rows + 65534) / 65535));
  if (plan.each == 32)
    piece_kernel<T, N, 32><<<grid, kThreads, 0, stream>>>(p, (int)plan.pieces, best, norms);
  else if (plan.each == 16)
    piece_kernel<T, N, 16><<<grid, kThreads, 0, stream>>>(p, (int)plan.pieces, best, norms);
  else
    piece_kernel<T, N, 8><<<grid, kThreads, 0, stream>>>(p, (int)plan.pieces, best, norms);
  return cudaGetLastError();
}

template <class T>
cudaError_t pieces_words(const SelectParams& p, const SelectPlan& plan, ScoreKey* best, float2* norms,
                         cudaStream_t stream) {
  const int w = word_bytes(reinterpret_cast<uintptr_t>(p.scores) | (unsigned long long)(p.seq_stride * sizeof(T)) |
                           (unsigned long long)(p.beam_stride * sizeof(T)));
  if (w == 16) return pieces_t<T, 16 / sizeof(T)>(p, plan, best, norms, stream);
  if (w >= 4) return pieces_t<T, 4 / sizeof(T)>(p, plan, best, norms, stream);
  return pieces_t<T, 1>(p, plan, best, norms, stream);
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

// Grid: pieces of a row x rows x states
__global__ void __launch_bounds__(kThreads) reorder_kernel(const __grid_constant__ ReorderParams p) {
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
  cudaError_t e = p.type == kF32   ? pieces_words<float>(p, plan, best, norms, stream)
                  : p.type == kF16 ? pieces_words<__half>(p, plan, best, norms, stream)
                                   : pieces_words<__nv_bfloat16>(p, plan, best, norms, stream);
  if (e != cudaSuccess) return e;
  e = allow_smem<sequence_kernel>();
  if (e != cudaSuccess) return e;
  sequence_kernel<<<(unsigned)p.sequences, kThreads, smem, stream>>>(p, (int)plan.pieces, best, norms);
  return cudaGetLastError();
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
  reorder_kernel<<<dim3((unsigned)(pieces < 4096 ? pieces : 4096), (unsigned)(rows < 65535 ? rows : 65535), (unsigned)count),
                   kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace hnsw
