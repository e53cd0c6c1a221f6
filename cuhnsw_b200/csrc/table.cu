// Rows of a table of embeddings looked up by number, and the gradient of the table.
//
//   lookup:  out[t] = scale * rows[ids[t]]
//   grad:    out[r] = scale * sum over the t with ids[t] = r of grad[t]
//
// An id outside 0..n-1 is an empty slot (a search writes -1 there): a row of zeros, and no gradient.
#include "common.cuh"
#include "table_common.cuh"

namespace hnsw {

namespace {

__device__ __forceinline__ long long id_at(const void* ids, int ids64, long long t) {
  return ids64 ? __ldg(static_cast<const long long*>(ids) + t) : (long long)__ldg(static_cast<const int*>(ids) + t);
}

// ---- lookup ---------------------------------------------------------------------------------------------------------

constexpr int kLookupThreads = 256;

// `lanes` threads take kRows tokens at once, so that kRows loads of each are in flight.  Bound: HBM bytes.
template <class T, int N, int kRows>
__global__ void __launch_bounds__(kLookupThreads) lookup_kernel(LookupParams p, int lanes) {
  const int group = threadIdx.x / lanes, lane = threadIdx.x % lanes, groups = kLookupThreads / lanes;
  const long long first = ((long long)blockIdx.x * groups + group) * kRows;
  if (first >= p.tokens) return;
  const T* rows = static_cast<const T*>(p.rows);
  T* out = static_cast<T*>(p.out);
  long long id[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    id[r] = first + r < p.tokens ? id_at(p.ids, p.ids64, first + r) : -1;
    if (id[r] >= p.n) id[r] = -1;
  }
  for (long long c = (long long)lane * N; c < p.d; c += (long long)lanes * N) {
    Vec<T, N> v[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (id[r] >= 0) {
        v[r] = load_vec<T, N>(rows + id[r] * p.row_stride + c);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[r].v[i] = from_f32<T>(0.0f);
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (first + r >= p.tokens) break;
      if (id[r] >= 0 && p.scale != 1.0f) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[r].v[i] = from_f32<T>(to_f32(v[r].v[i]) * p.scale);
      }
      store_vec<T, N>(out + (first + r) * p.d + c, v[r]);
    }
  }
}

template <class T, int N>
cudaError_t lookup_t(const LookupParams& p, cudaStream_t stream) {
  const int lanes = next_pow2((p.d + N - 1) / N, kLookupThreads);
  const int groups = kLookupThreads / lanes;
  // four rows at a time, unless there are too few tokens to give every SM work
  const bool many = p.tokens > (long long)4 * groups * kSMs;
  const long long per = (many ? 4 : 1) * groups;
  const long long blocks = (p.tokens + per - 1) / per;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  if (many)
    lookup_kernel<T, N, 4><<<(unsigned)blocks, kLookupThreads, 0, stream>>>(p, lanes);
  else
    lookup_kernel<T, N, 1><<<(unsigned)blocks, kLookupThreads, 0, stream>>>(p, lanes);
  return cudaGetLastError();
}

template <class T>
cudaError_t lookup_words(const LookupParams& p, cudaStream_t stream) {
  const int w = word_bytes(reinterpret_cast<uintptr_t>(p.rows) | reinterpret_cast<uintptr_t>(p.out) |
                           (unsigned long long)(p.row_stride * sizeof(T)) | (unsigned long long)(p.d * sizeof(T)));
  if (w == 16) return lookup_t<T, 16 / sizeof(T)>(p, stream);
  if (w == 8) return lookup_t<T, 8 / sizeof(T)>(p, stream);
  if (w == 4) return lookup_t<T, 4 / sizeof(T)>(p, stream);
  return lookup_t<T, 1>(p, stream);
}

// ---- gradient: the tokens sorted by id ------------------------------------------------------------------------------

// A least-significant-digit radix sort of (id, token): stable, so the tokens of a row stay in their order and its sum does
// not depend on the launch.  Ids outside the table become n, the largest key.
constexpr int kOneThreads = 1024;       // one CTA sorts up to kOneMost tokens in shared memory
constexpr int kOneItems = 16;
constexpr int kOneMost = kOneThreads * kOneItems;
constexpr int kTileThreads = 256;       // more: tiles of kTile tokens, one launch per step
constexpr int kTileItems = 16;
constexpr int kTile = kTileThreads * kTileItems;
constexpr int kMaxDigit = 8;

struct SortPlan {
  int bits, passes, digit;
};
SortPlan sort_plan(long long n) {
  SortPlan s;
  s.bits = 1;
  while (s.bits < 32 && (n >> s.bits) > 0) ++s.bits;  // keys 0..n
  s.passes = (s.bits + kMaxDigit - 1) / kMaxDigit;
  s.digit = (s.bits + s.passes - 1) / s.passes;
  return s;
}

__device__ __forceinline__ unsigned key_at(const LookupGradParams& p, long long t) {
  const long long id = id_at(p.ids, p.ids64, t);
  return id < 0 || id >= p.n ? (unsigned)p.n : (unsigned)id;
}

// Rank of each of a warp's keys (lane l holds items l, 32 + l, ..) among the earlier keys of the warp with the same
// digit; counts[digit] ends as the warp's number of keys with that digit.
template <int Items>
__device__ __forceinline__ void warp_ranks(const unsigned (&key)[Items], int shift, unsigned mask, int valid,
                                           unsigned short* counts, unsigned (&rank)[Items]) {
  const unsigned earlier = (1u << lane_id()) - 1;
#pragma unroll
  for (int i = 0; i < Items; ++i) {
    if (i * 32 >= valid) break;
    const bool live = i * 32 + lane_id() < valid;
    const unsigned digit = (key[i] >> shift) & mask;
    const unsigned peers = __match_any_sync(FULL, live ? digit : 0xffffffffu);
    const unsigned before = live ? counts[digit] : 0;
    __syncwarp();
    if (live && (peers & earlier) == 0) counts[digit] = (unsigned short)(before + __popc(peers));
    __syncwarp();
    rank[i] = before + __popc(peers & earlier);
  }
}

// Exclusive sum of one value per thread over the CTA.
template <int Threads>
__device__ __forceinline__ unsigned block_exclusive(unsigned x, unsigned* scratch /* Threads / 32 */) {
  const int lane = lane_id(), warp = threadIdx.x >> 5;
  unsigned sum = x;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const unsigned y = __shfl_up_sync(FULL, sum, off);
    if (lane >= off) sum += y;
  }
  if (lane == 31) scratch[warp] = sum;
  __syncthreads();
  unsigned before = 0;
  for (int w = 0; w < warp; ++w) before += scratch[w];
  __syncthreads();
  return before + sum - x;
}

// Zeros in all of `out`, by the CTAs [first, gridDim.x) of a launch.
__device__ __forceinline__ void zero_out(const LookupGradParams& p, int first) {
  unsigned char* out = static_cast<unsigned char*>(p.out);
  const unsigned long long bytes = (unsigned long long)p.n * p.d * (p.out_type == kF32 ? 4 : 2);
  // whole words of 16 bytes, and single bytes before and behind them
  const unsigned long long head = min(bytes, (unsigned long long)(-reinterpret_cast<uintptr_t>(out) & 15));
  const unsigned long long words = (bytes - head) / 16, tail = (bytes - head) % 16;
  if ((int)blockIdx.x == first) {
    if (threadIdx.x < head) out[threadIdx.x] = 0;
    if (threadIdx.x < tail) out[head + words * 16 + threadIdx.x] = 0;
  }
  const unsigned long long step = (unsigned long long)(gridDim.x - first) * blockDim.x;
  uint4* to = reinterpret_cast<uint4*>(out + head);
  for (unsigned long long at = (unsigned long long)(blockIdx.x - first) * blockDim.x + threadIdx.x; at < words; at += step)
    __stcs(to + at, make_uint4(0, 0, 0, 0));
}

// CTA 0 sorts all tokens in shared memory; the others meanwhile write the zeros of the rows that nobody looked up.
__global__ void __launch_bounds__(kOneThreads) sort_one_kernel(LookupGradParams p, SortPlan plan, unsigned* keys_out,
                                                               unsigned* tokens_out, unsigned* joins) {
  if (blockIdx.x > 0) {
    zero_out(p, 1);
    return;
  }
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int kWarps = kOneThreads / 32;
  const int digits = 1 << plan.digit, count = (int)p.tokens;
  const int items = (count + kOneThreads - 1) / kOneThreads;
  unsigned* keys = reinterpret_cast<unsigned*>(smem);
  unsigned short* places = reinterpret_cast<unsigned short*>(keys + items * kOneThreads);
  unsigned short* counts = places + items * kOneThreads;
  __shared__ unsigned scratch[kWarps];
  const int warp = threadIdx.x >> 5, lane = lane_id();
  const int begin = min(warp * items * 32, count), valid = min(items * 32, count - begin);
  if (threadIdx.x == 0) *joins = 0;
  for (int t = threadIdx.x; t < count; t += kOneThreads) {
    keys[t] = key_at(p, t);
    places[t] = (unsigned short)t;
  }
  for (int pass = 0; pass < plan.passes; ++pass) {
    const int shift = pass * plan.digit;
    for (int i = threadIdx.x; i < kWarps * digits; i += kOneThreads) counts[i] = 0;
    __syncthreads();
    unsigned key[kOneItems], rank[kOneItems];
    unsigned short place[kOneItems];
#pragma unroll
    for (int i = 0; i < kOneItems; ++i) {
      if (i * 32 + lane < valid) {
        key[i] = keys[begin + i * 32 + lane];
        place[i] = places[begin + i * 32 + lane];
      }
    }
    warp_ranks<kOneItems>(key, shift, digits - 1, valid, counts + warp * digits, rank);
    __syncthreads();
    unsigned total = 0;
    if (threadIdx.x < digits) {
      for (int w = 0; w < kWarps; ++w) {
        const unsigned c = counts[w * digits + threadIdx.x];
        counts[w * digits + threadIdx.x] = (unsigned short)total;
        total += c;
      }
    }
    const unsigned base = block_exclusive<kOneThreads>(total, scratch);
    if (threadIdx.x < digits)
      for (int w = 0; w < kWarps; ++w) counts[w * digits + threadIdx.x] += (unsigned short)base;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOneItems; ++i) {
      if (i * 32 + lane < valid) {
        const unsigned at = counts[warp * digits + ((key[i] >> shift) & (digits - 1))] + rank[i];
        if (pass + 1 < plan.passes) {
          keys[at] = key[i];
          places[at] = place[i];
        } else {
          keys_out[at] = key[i];
          tokens_out[at] = place[i];
        }
      }
    }
    __syncthreads();
  }
}

// Tokens of each digit in each tile, digit by digit: counts[digit * tiles + tile].  In the first pass the CTAs behind the
// tiles write the zeros.
__global__ void __launch_bounds__(kTileThreads) sort_count_kernel(LookupGradParams p, const unsigned* keys, int shift,
                                                                  int digits, int tiles, unsigned* counts,
                                                                  unsigned* joins) {
  if ((int)blockIdx.x >= tiles) {
    zero_out(p, tiles);
    return;
  }
  __shared__ unsigned bins[1 << kMaxDigit];
  for (int i = threadIdx.x; i < digits; i += kTileThreads) bins[i] = 0;
  if (joins && blockIdx.x == 0 && threadIdx.x == 0) *joins = 0;
  __syncthreads();
  const long long begin = (long long)blockIdx.x * kTile;
  const int valid = (int)min((long long)kTile, p.tokens - begin);
  for (int from = threadIdx.x & ~31; from < valid; from += kTileThreads) {
    const int i = from + lane_id();
    const bool live = i < valid;
    const unsigned key = !live ? 0 : keys ? keys[begin + i] : key_at(p, begin + i);
    const unsigned digit = live ? (key >> shift) & (digits - 1) : 0xffffffffu;
    // one addition for all lanes with the same digit: a frequent token would serialise them
    const unsigned peers = __match_any_sync(FULL, digit);
    if (live && (peers & ((1u << lane_id()) - 1)) == 0) atomicAdd(bins + digit, __popc(peers));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < digits; i += kTileThreads) counts[(size_t)i * tiles + blockIdx.x] = bins[i];
}

// Exclusive sum of all counts, by one CTA.
__global__ void __launch_bounds__(kOneThreads) sort_scan_kernel(unsigned* counts, long long total) {
  __shared__ unsigned scratch[kOneThreads / 32];
  __shared__ unsigned carry;
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  constexpr int kEach = 16;
  for (long long begin = 0; begin < total; begin += kOneThreads * kEach) {
    const long long mine = begin + (long long)threadIdx.x * kEach;
    unsigned c[kEach], sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      c[i] = mine + i < total ? counts[mine + i] : 0;
      sum += c[i];
    }
    unsigned before = block_exclusive<kOneThreads>(sum, scratch) + carry;
    const unsigned after = before + sum;
    __syncthreads();
    if (threadIdx.x == kOneThreads - 1) carry = after;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (mine + i < total) counts[mine + i] = before;
      before += c[i];
    }
    __syncthreads();
  }
}

// Every tile's tokens to their places.
__global__ void __launch_bounds__(kTileThreads) sort_place_kernel(LookupGradParams p, const unsigned* keys,
                                                                  const unsigned* tokens, int shift, int digits,
                                                                  int tiles, const unsigned* counts, unsigned* keys_out,
                                                                  unsigned* tokens_out) {
  constexpr int kWarps = kTileThreads / 32;
  __shared__ unsigned short warp_counts[kWarps << kMaxDigit];
  __shared__ unsigned bases[kWarps << kMaxDigit];
  const int warp = threadIdx.x >> 5, lane = lane_id();
  for (int i = threadIdx.x; i < kWarps * digits; i += kTileThreads) warp_counts[i] = 0;
  __syncthreads();
  const long long tile_begin = (long long)blockIdx.x * kTile;
  const long long begin = min(tile_begin + warp * 32 * kTileItems, p.tokens);
  const int valid = (int)min((long long)(32 * kTileItems), p.tokens - begin);
  unsigned key[kTileItems], token[kTileItems], rank[kTileItems];
#pragma unroll
  for (int i = 0; i < kTileItems; ++i) {
    if (i * 32 + lane < valid) {
      const long long at = begin + i * 32 + lane;
      key[i] = keys ? keys[at] : key_at(p, at);
      token[i] = tokens ? tokens[at] : (unsigned)at;
    }
  }
  warp_ranks<kTileItems>(key, shift, digits - 1, valid, warp_counts + warp * digits, rank);
  __syncthreads();
  for (int i = threadIdx.x; i < digits; i += kTileThreads) {
    unsigned base = counts[(size_t)i * tiles + blockIdx.x];
    for (int w = 0; w < kWarps; ++w) {
      bases[w * digits + i] = base;
      base += warp_counts[w * digits + i];
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kTileItems; ++i) {
    if (i * 32 + lane < valid) {
      const unsigned at = bases[warp * digits + ((key[i] >> shift) & (digits - 1))] + rank[i];
      keys_out[at] = key[i];
      tokens_out[at] = token[i];
    }
  }
}

// ---- gradient: sums over the sorted tokens --------------------------------------------------------------------------

// The sorted tokens are cut into chunks of equal length, whatever rows they belong to: a frequent token makes no CTA's work
// longer.  A row whose tokens all lie in one chunk is written there; of a row that crosses a border each chunk leaves a
// partial sum in fp32 (heads: of the row that the chunk before began; tails: of the row that goes on in the next one), and
// join_kernel adds those up.
constexpr int kSumThreads = 256;
constexpr int kInFlight = 8;

struct SumPlan {
  int chunk;         // tokens
  long long chunks;
};
SumPlan sum_plan(long long tokens, long long d) {
  SumPlan s;
  // about 2048 values per SM and chunk of 64 tokens keep all SMs busy; short batches take shorter chunks
  s.chunk = 64;
  while (s.chunk > 8 && tokens / s.chunk * d < (long long)kSMs * 4096) s.chunk /= 2;
  s.chunks = (tokens + s.chunk - 1) / s.chunk;
  return s;
}

template <class G, class O, int N>
__device__ __forceinline__ void write_row(const LookupGradParams& p, unsigned row, long long c, const float (&sum)[N]) {
  O* at = static_cast<O*>(p.out) + (long long)row * p.d + c;
  O v[N];
  if (p.accumulate) load_many<O, N>(at, v);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = from_f32<O>(p.accumulate ? to_f32(v[i]) + sum[i] * p.scale : sum[i] * p.scale);
  store_many<O, N>(at, v);
}

template <class G, class O, int N>
__global__ void __launch_bounds__(kSumThreads) sum_kernel(LookupGradParams p, SumPlan plan, const unsigned* keys,
                                                          const unsigned* tokens, float* heads, float* tails,
                                                          unsigned* joins, unsigned* join_list, int lanes) {
  const int group = threadIdx.x / lanes, lane = threadIdx.x % lanes, groups = kSumThreads / lanes;
  const long long chunk = (long long)blockIdx.x * groups + group;
  if (chunk >= plan.chunks) return;
  const long long begin = chunk * plan.chunk, end = min(begin + plan.chunk, p.tokens);
  const long long c = ((long long)blockIdx.y * lanes + lane) * N;
  if (c >= p.d) return;
  const unsigned none = (unsigned)p.n;
  const G* grad = static_cast<const G*>(p.grad);
  const unsigned before = begin > 0 ? keys[begin - 1] : none, after = end < p.tokens ? keys[end] : none;
  unsigned row = keys[begin];
  bool first = true;  // the row that the chunk begins with
  float sum[N];
#pragma unroll
  for (int i = 0; i < N; ++i) sum[i] = 0.0f;
  auto finish = [&](bool last) {
    if (row == none) return;
    float* partial = nullptr;
    if (first && row == before)
      partial = heads + chunk * p.d + c;
    else if (last && row == after)
      partial = tails + chunk * p.d + c;
    if (partial) {
      store_many<float, N>(partial, sum);
      if (last && row == after && !(first && row == before) && c == 0) join_list[atomicAdd(joins, 1u)] = (unsigned)chunk;
    } else {
      write_row<G, O, N>(p, row, c, sum);
    }
  };
  for (long long t = begin; t < end; t += kInFlight) {
    unsigned key[kInFlight];
    Vec<G, N> v[kInFlight];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      key[i] = t + i < end ? keys[t + i] : none;
      if (key[i] != none) v[i] = load_stream<G, N>(grad + (long long)tokens[t + i] * p.grad_stride + c);
    }
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      if (t + i >= end) break;
      if (key[i] != row) {
        finish(false);
        row = key[i];
        first = false;
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] = 0.0f;
      }
      if (row == none) return;  // nothing but empty slots from here on
#pragma unroll
      for (int j = 0; j < N; ++j) sum[j] += to_f32(v[i].v[j]);
    }
  }
  finish(true);
}

// Rows that cross borders of chunks: 8 warps add up an eighth of the partial sums each.
constexpr int kJoinWarps = 8;
template <class G, class O>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(LookupGradParams p, SumPlan plan, const unsigned* keys,
                                                               const float* heads, const float* tails,
                                                               const unsigned* joins, const unsigned* join_list) {
  __shared__ float sums[kJoinWarps][32];
  const int warp = threadIdx.x >> 5, lane = lane_id();
  const unsigned count = *joins;
  const long long c = (long long)blockIdx.y * 32 + lane;
  for (unsigned i = blockIdx.x; i < count; i += gridDim.x) {
    const long long chunk = join_list[i];
    const unsigned row = keys[(chunk + 1) * plan.chunk];
    // the last chunk that the row reaches: its first key is the row's
    long long low = chunk + 1, high = plan.chunks - 1;
    while (low < high) {
      const long long mid = (low + high + 1) / 2;
      if (keys[mid * plan.chunk] == row)
        low = mid;
      else
        high = mid - 1;
    }
    const long long parts = low - chunk + 1;  // one tail, the rest heads
    const long long each = (parts + kJoinWarps - 1) / kJoinWarps;
    float sum = 0.0f;
    if (c < p.d) {
      const long long to = min(parts, (warp + 1) * each);
#pragma unroll 8
      for (long long k = warp * each; k < to; ++k) sum += (k == 0 ? tails : heads)[(chunk + k) * p.d + c];
    }
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && c < p.d) {
      float total[1] = {sums[0][lane]};
#pragma unroll
      for (int w = 1; w < kJoinWarps; ++w) total[0] += sums[w][lane];
      write_row<G, O, 1>(p, row, c, total);
    }
    __syncthreads();
  }
}

struct GradSpace {
  unsigned* keys[2];
  unsigned* tokens[2];
  unsigned* counts;
  unsigned* joins;
  unsigned* join_list;
  float* heads;
  float* tails;
  size_t bytes;
};
GradSpace grad_space(long long tokens, long long n, long long d, void* base) {
  GradSpace s;
  unsigned char* at = static_cast<unsigned char*>(base);
  size_t used = 0;
  auto take = [&](long long count) {
    unsigned char* here = at + used;
    used += ((size_t)count * 4 + 255) / 256 * 256;
    return here;
  };
  const SumPlan sums = sum_plan(tokens, d);
  const SortPlan plan = sort_plan(n);
  const bool one = tokens <= kOneMost;
  for (int i = 0; i < 2; ++i) {
    s.keys[i] = reinterpret_cast<unsigned*>(take(one && i ? 0 : tokens));
    s.tokens[i] = reinterpret_cast<unsigned*>(take(one && i ? 0 : tokens));
  }
  s.counts = reinterpret_cast<unsigned*>(take(one ? 0 : ((tokens + kTile - 1) / kTile) << plan.digit));
  s.joins = reinterpret_cast<unsigned*>(take(1));
  s.join_list = reinterpret_cast<unsigned*>(take(sums.chunks));
  s.heads = reinterpret_cast<float*>(take(sums.chunks * d));
  s.tails = reinterpret_cast<float*>(take(sums.chunks * d));
  s.bytes = used;
  return s;
}

template <class G, class O, int N>
cudaError_t sum_t(const LookupGradParams& p, const SumPlan& plan, const GradSpace& s, int at, cudaStream_t stream) {
  const int lanes = next_pow2((p.d + N - 1) / N, kSumThreads);
  const int groups = kSumThreads / lanes;
  const long long blocks = (plan.chunks + groups - 1) / groups, columns = (p.d + (long long)lanes * N - 1) / ((long long)lanes * N);
  if (blocks > 0x7fffffffll || columns > 65535) return cudaErrorInvalidValue;
  sum_kernel<G, O, N><<<dim3((unsigned)blocks, (unsigned)columns), kSumThreads, 0, stream>>>(
    p, plan, s.keys[at], s.tokens[at], s.heads, s.tails, s.joins, s.join_list, lanes);
  return cudaGetLastError();
}

template <class G, class O>
cudaError_t grad_t(const LookupGradParams& p, cudaStream_t stream) {
  const SumPlan plan = sum_plan(p.tokens, p.d);
  const SortPlan sort = sort_plan(p.n);
  const GradSpace s = grad_space(p.tokens, p.n, p.d, p.workspace);
  const int zero_blocks = p.accumulate ? 0 : kSMs;
  int at = 0;
  if (p.tokens <= kOneMost) {
    const int items = (int)((p.tokens + kOneThreads - 1) / kOneThreads);
    const size_t smem = (size_t)items * kOneThreads * 6 + (size_t)(kOneThreads / 32) * (1 << sort.digit) * 2;
    cudaError_t e = allow_smem<sort_one_kernel>();
    if (e != cudaSuccess) return e;
    sort_one_kernel<<<1 + zero_blocks, kOneThreads, smem, stream>>>(p, sort, s.keys[0], s.tokens[0], s.joins);
  } else {
    const long long tiles = (p.tokens + kTile - 1) / kTile;
    const int digits = 1 << sort.digit;
    for (int pass = 0; pass < sort.passes; ++pass) {
      const unsigned* keys = pass ? s.keys[at] : nullptr;
      const unsigned* tokens = pass ? s.tokens[at] : nullptr;
      const int to = pass ? 1 - at : 0;
      sort_count_kernel<<<(unsigned)(tiles + (pass ? 0 : 4 * zero_blocks)), kTileThreads, 0, stream>>>(
        p, keys, pass * sort.digit, digits, (int)tiles, s.counts, pass ? nullptr : s.joins);
      sort_scan_kernel<<<1, kOneThreads, 0, stream>>>(s.counts, tiles * digits);
      sort_place_kernel<<<(unsigned)tiles, kTileThreads, 0, stream>>>(p, keys, tokens, pass * sort.digit, digits,
                                                                     (int)tiles, s.counts, s.keys[to], s.tokens[to]);
      at = to;
    }
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int w = word_bytes(reinterpret_cast<uintptr_t>(p.grad) | (unsigned long long)(p.grad_stride * sizeof(G)) |
                           (unsigned long long)(p.d * sizeof(G)));
  const int to = word_bytes(reinterpret_cast<uintptr_t>(p.out)) / (int)sizeof(O) * (int)sizeof(G);
  if (w == 16 && to * sizeof(O) >= 16 * sizeof(G))
    e = sum_t<G, O, 16 / sizeof(G)>(p, plan, s, at, stream);
  else if (w >= 8 && to >= 8)
    e = sum_t<G, O, 8 / sizeof(G)>(p, plan, s, at, stream);
  else if (w >= 4 && to >= 4)
    e = sum_t<G, O, 4 / sizeof(G)>(p, plan, s, at, stream);
  else
    e = sum_t<G, O, 1>(p, plan, s, at, stream);
  if (e != cudaSuccess || plan.chunks < 2) return e;
  const long long columns = (p.d + 31) / 32;
  if (columns > 65535) return cudaErrorInvalidValue;
  const long long rows = plan.chunks < 4 * kSMs ? plan.chunks : 4 * kSMs;
  join_kernel<G, O><<<dim3((unsigned)rows, (unsigned)columns), kJoinWarps * 32, 0, stream>>>(
    p, plan, s.keys[at], s.heads, s.tails, s.joins, s.join_list);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_lookup(const LookupParams& p, cudaStream_t stream) {
  if (p.tokens <= 0 || p.d <= 0) return cudaSuccess;
  if (p.type == kF32) return lookup_words<float>(p, stream);
  if (p.type == kF16) return lookup_words<__half>(p, stream);
  return lookup_words<__nv_bfloat16>(p, stream);
}

size_t lookup_grad_workspace(long long tokens, long long n, long long d) {
  return tokens <= 0 || n <= 0 || d <= 0 ? 0 : grad_space(tokens, n, d, nullptr).bytes;
}

cudaError_t launch_lookup_grad(const LookupGradParams& p, cudaStream_t stream) {
  if (p.n <= 0 || p.d <= 0) return cudaSuccess;
  if (p.tokens <= 0) {
    if (p.accumulate) return cudaSuccess;
    return cudaMemsetAsync(p.out, 0, (size_t)p.n * p.d * type_size(p.out_type), stream);
  }
  if (p.type == kF32) return grad_t<float, float>(p, stream);
  if (p.type == kF16)
    return p.out_type == kF32 ? grad_t<__half, float>(p, stream) : grad_t<__half, __half>(p, stream);
  return p.out_type == kF32 ? grad_t<__nv_bfloat16, float>(p, stream) : grad_t<__nv_bfloat16, __nv_bfloat16>(p, stream);
}

}  // namespace hnsw
