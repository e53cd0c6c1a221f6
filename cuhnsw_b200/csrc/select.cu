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

// Candidates of a CTA in shared memory, in any order; `sort` puts them in descending order.
template <class Key>
struct Pool {
  Key* keys;
  int* count;
  int capacity;  // a power of two

  __device__ void push(const Key& k) { keys[atomicAdd(count, 1)] = k; }

  // Bitonic over the smallest power of two that holds them; all threads.
  __device__ void sort() {
    __syncthreads();
    const int held = *count;
    int size = 2;
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
// into a pool, the pool in order.  Also the piece's largest score and its sum of exponentials.
constexpr int kPoolScores = 2048;

template <class T, int N, int kEach>
__global__ void __launch_bounds__(kThreads) piece_kernel(SelectParams p, int pieces, ScoreKey* best, float2* norms) {
  __shared__ ScoreKey pool_keys[kPoolScores];
  __shared__ int pool_count;
  __shared__ ScoreKey firsts[kThreads];
  __shared__ float warp_max[kThreads / 32], warp_sum[kThreads / 32];
  const int warp = threadIdx.x >> 5, lane = lane_id();
  const long long row = blockIdx.y + (long long)blockIdx.z * 65535;
  if (row >= p.sequences * p.beams) return;
  const long long seq = row / p.beams, beam = row % p.beams;
  const T* scores = static_cast<const T*>(p.scores) + seq * p.seq_stride + beam * p.beam_stride;
  const long long begin = (long long)blockIdx.x * kThreads * kEach;
  float x[kEach];
#pragma unroll
  for (int i = 0; i < kEach; i += N) {
    const long long at = begin + (long long)(i / N * kThreads + threadIdx.x) * N;
    if (at + N <= p.vocabulary) {
      const Vec<T, N> v = load_stream<T, N>(scores + at);
#pragma unroll
      for (int j = 0; j < N; ++j) x[i + j] = to_f32(v.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) x[i + j] = at + j < p.vocabulary ? to_f32(scores[at + j]) : -INFINITY;
    }
  }
  auto place = [&](int i) { return (unsigned)(begin + (long long)(i / N * kThreads + threadIdx.x) * N + i % N); };
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kEach; ++i) top = fmaxf(top, x[i]);
  ScoreKey mine = 0;
#pragma unroll
  for (int i = kEach - 1; i >= 0; --i)
    if (x[i] == top) mine = score_key(top, place(i));
  if (p.log_softmax) {
    float most = top;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(FULL, most, off));
    if (lane == 0) warp_max[warp] = most;
    __syncthreads();
    most = -FLT_MAX;  // (of a row of -inf the exponentials are zeros)
    for (int w = 0; w < kThreads / 32; ++w) most = fmaxf(most, warp_max[w]);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += __expf(x[i] - most);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(FULL, sum, off);
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      float all = 0.0f;
      for (int w = 0; w < kThreads / 32; ++w) all += warp_sum[w];
      norms[row * pieces + blockIdx.x] = make_float2(most, all);
    }
  }
  // the bound: groups of `lanes` threads
  int lanes = kThreads;
  while (lanes > 1 && kThreads / lanes < p.keep) lanes >>= 1;
  ScoreKey bound = mine;
  for (int off = 1; off < lanes && off < 32; off <<= 1) {
    const ScoreKey other = shfl64(bound, lane ^ off);
    bound = other > bound ? other : bound;
  }
  firsts[threadIdx.x] = bound;
  if (threadIdx.x == 0) pool_count = 0;
  __syncthreads();
  const int stride = min(lanes, 32);
  if (lanes > 32) {
    // a group is several warps
    ScoreKey of_group = 0;
    const int from = threadIdx.x / lanes * lanes;
    for (int i = from; i < from + lanes; i += 32) of_group = firsts[i] > of_group ? firsts[i] : of_group;
    bound = of_group;
    __syncthreads();
    firsts[threadIdx.x] = bound;
    __syncthreads();
  }
  // the smallest over the groups
  ScoreKey least = ~0ull;
  for (int i = lane * stride; i < kThreads; i += 32 * stride) least = firsts[i] < least ? firsts[i] : least;
  for (int off = 16; off > 0; off >>= 1) {
    const ScoreKey other = shfl64(least, lane ^ off);
    least = other < least ? other : least;
  }
  int passing = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const ScoreKey k = score_key(x[i], place(i));
    passing += k != 0 && k >= least;
  }
  Pool<ScoreKey> pool{pool_keys, &pool_count, kPoolScores};
  if (__syncthreads_count(passing > 0) == 0) {
    // nothing to choose from
  } else if (__syncthreads_or(passing > kPoolScores / kThreads) == 0) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const ScoreKey k = score_key(x[i], place(i));
      if (k != 0 && k >= least) pool.push(k);
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < kEach; ++i) {
      pool.make_room(p.keep, least);
      float xi = x[0];
#pragma unroll
      for (int j = 1; j < kEach; ++j) xi = j == i ? x[j] : xi;
      const ScoreKey k = score_key(xi, place(i));
      if (k != 0 && k >= least) pool.push(k);
    }
  }
  pool.sort();
  ScoreKey* to = best + (row * pieces + blockIdx.x) * p.keep;
  const int held = min(pool_count, p.keep);
  for (int i = threadIdx.x; i < p.keep; i += kThreads) to[i] = i < held ? pool_keys[i] : 0;
}

// ---- a sequence -----------------------------------------------------------------------------------------------------

constexpr int kPoolTotals = 2048;

// One CTA per sequence: all pieces' lists in order of rank, so that the best of every list come first and the bound rises
// at once.
__global__ void __launch_bounds__(kThreads) sequence_kernel(SelectParams p, int pieces, const ScoreKey* best,
                                                            const float2* norms) {
  extern __shared__ __align__(16) unsigned char smem[];
  TotalKey* pool_keys = reinterpret_cast<TotalKey*>(smem);
  double* offsets = reinterpret_cast<double*>(pool_keys + kPoolTotals);  // what a beam's scores are raised by
  __shared__ int pool_count;
  const int lane = lane_id(), warp = threadIdx.x >> 5;
  const long long seq = blockIdx.x;
  const int beams = (int)p.beams;
  if (threadIdx.x == 0) pool_count = 0;
  for (int b = warp; b < beams; b += kThreads / 32) {
    double offset = p.totals ? (double)p.totals[seq * beams + b] : 0.0;
    if (p.log_softmax) {
      const float2* of_row = norms + (seq * beams + b) * pieces;
      float most = -FLT_MAX;
      for (int i = lane; i < pieces; i += 32) most = fmaxf(most, of_row[i].x);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor_sync(FULL, most, off));
      double sum = 0.0;
      for (int i = lane; i < pieces; i += 32) sum += of_row[i].y * exp((double)of_row[i].x - (double)most);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(FULL, sum, off);
      offset -= (double)most + log(sum);
    }
    if (lane == 0) offsets[b] = offset;
  }
  __syncthreads();
  Pool<TotalKey> pool{pool_keys, &pool_count, kPoolTotals};
  TotalKey least = {0, 0, 0};
  const long long lists = (long long)beams * pieces, total = lists * p.keep;
  const ScoreKey* mine = best + seq * total;
  for (long long begin = 0; begin < total; begin += kThreads) {
    pool.make_room(p.keep, least);
    const long long i = begin + threadIdx.x;
    if (i < total) {
      const long long list = i % lists, rank = i / lists;
      const ScoreKey k = mine[list * p.keep + rank];
      if (k != 0) {
        const unsigned beam = (unsigned)(list / pieces);
        const double value = offsets[beam] + (double)key_score(k);
        if (value > -INFINITY) {
          const TotalKey key = {d2ord(value), key_place(k), beam};
          if (none(least) || !above(least, key)) pool.push(key);
        }
      }
    }
  }
  pool.sort();
  const int found = min(pool_count, p.keep);
  for (int i = threadIdx.x; i < p.keep; i += kThreads) {
    const TotalKey k = pool_keys[min(i, kPoolTotals - 1)];
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
