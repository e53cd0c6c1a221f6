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
  return ids64 ? static_cast<const long long*>(ids)[t] : (long long)static_cast<const int*>(ids)[t];
}

// ---- lookup ---------------------------------------------------------------------------------------------------------

constexpr int kLookupThreads = 256;

// `lanes` threads take kRows tokens at once and kAt words of each, so that so many loads of each are in flight.  Bound: HBM bytes
// (100 000 rows of 50 floats out of 1 183 514 in 10 us, 4.1 TB/s of sectors of 32 bytes), of few tokens the launch (3 us).
template <class T, int N, int kRows, int kAt>
__global__ void __launch_bounds__(kLookupThreads) lookup_kernel(LookupParams p, int lanes) {
  const int group = threadIdx.x / lanes, lane = threadIdx.x % lanes, groups = kLookupThreads / lanes;
  next_launch_may_start();
  wait_for_launch_before();
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
  const int step = lanes * N, d = (int)p.d;
  for (int begin = lane * N; begin < d; begin += kAt * step) {
    Vec<T, N> v[kRows][kAt];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
      for (int k = 0; k < kAt; ++k) {
        const int c = begin + k * step;
        if (id[r] >= 0 && c < d) {
          v[r][k] = load_vec<T, N>(rows + id[r] * p.row_stride + c);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) v[r][k].v[i] = from_f32<T>(0.0f);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (first + r >= p.tokens) break;
#pragma unroll
      for (int k = 0; k < kAt; ++k) {
        const int c = begin + k * step;
        if (c >= d) break;
        if (id[r] >= 0 && p.scale != 1.0f) {
#pragma unroll
          for (int i = 0; i < N; ++i) v[r][k].v[i] = from_f32<T>(to_f32(v[r][k].v[i]) * p.scale);
        }
        store_vec<T, N>(out + (first + r) * p.d + c, v[r][k]);
      }
    }
  }
}

template <class T, int N>
cudaError_t lookup_t(const LookupParams& p, cudaStream_t stream) {
  // narrow words: four of each row
  constexpr int kAt = N * sizeof(T) >= 8 ? 1 : 4;
  const int lanes = next_pow2((p.d + kAt * N - 1) / (kAt * N), kLookupThreads);
  const int groups = kLookupThreads / lanes;
  // Four rows at a time, unless there are too few tokens to give every SM work.  (50 000 rows of 1024 bfloat16 30 us, one at a
  // time 48; 8 of 2048 3.4 us, one at a time 2.9.)
  const bool many = p.tokens > (long long)4 * groups * kSMs;
  const long long per = (many ? 4 : 1) * groups;
  const long long blocks = (p.tokens + per - 1) / per;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  if (many)
    return launch_early(lookup_kernel<T, N, 4, kAt>, dim3((unsigned)blocks), kLookupThreads, 0, stream, p, lanes);
  return launch_early(lookup_kernel<T, N, 1, kAt>, dim3((unsigned)blocks), kLookupThreads, 0, stream, p, lanes);
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

// Tokens sorted by id, those of a row in their order, so that its sum does not depend on the launch.  Ids outside the table
// become n, the largest key.  The launches that sort are short chains of dependent steps; on the SMs beside them the zeros of the
// rows without tokens are written (`zeros`: that part of `out`, by the CTAs behind `first`).

struct ZeroPart {
  int first;                          // CTAs from here on, kZeroWords each
  unsigned long long begin, words;    // of 16 bytes, from the first 16-byte boundary in `out`
  unsigned char* out;
  unsigned long long bytes;           // of all of `out`
};

// Many CTAs with a few words each: 1 GB in 147 us; 592 CTAs that go through it in strides take 174.
constexpr int kZeroThreads = 256;
constexpr int kZeroWords = 4 * kZeroThreads;

__device__ __forceinline__ void write_zeros(const ZeroPart& z) {
  // whole words of 16 bytes, and with the first ones single bytes before and behind them all
  const unsigned long long head = min(z.bytes, (unsigned long long)(-reinterpret_cast<uintptr_t>(z.out) & 15));
  if ((int)blockIdx.x == z.first && z.begin == 0) {
    const unsigned long long all = (z.bytes - head) / 16, tail = (z.bytes - head) % 16;
    if (threadIdx.x < head) z.out[threadIdx.x] = 0;
    if (threadIdx.x < tail) z.out[head + all * 16 + threadIdx.x] = 0;
  }
  uint4* to = reinterpret_cast<uint4*>(z.out + head) + z.begin;
  const unsigned long long at = (unsigned long long)(blockIdx.x - z.first) * kZeroWords + threadIdx.x;
#pragma unroll
  for (int i = 0; i < kZeroWords / kZeroThreads; ++i)
    if (at + i * kZeroThreads < z.words) to[at + i * kZeroThreads] = make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ unsigned key_at(const LookupGradParams& p, long long t) {
  const long long id = id_at(p.ids, p.ids64, t);
  return id < 0 || id >= p.n ? (unsigned)p.n : (unsigned)id;
}

// Up to kRankMost tokens: every token's place is the number of smaller keys and of equal ones before it, counted against all
// tokens: no pass depends on another one.  (The whole gradient, 64 floats a row: 4096 tokens 24 us, by digits 29; 6000 tokens 29
// and 30; 8192 tokens 40 and 32.)
constexpr int kRankMost = 6144;
constexpr int kRankThreads = kZeroThreads;
constexpr int kRankTokens = 64;                                // of a CTA
constexpr int kRankShares = kRankThreads / kRankTokens;        // threads that share a token
constexpr int kRankTile = 2048;                                // keys in shared memory at a time

__global__ void __launch_bounds__(kRankThreads) sort_rank_kernel(LookupGradParams p, ZeroPart zeros, uint2* sorted,
                                                                 unsigned* joins) {
  next_launch_may_start();
  wait_for_launch_before();
  if ((int)blockIdx.x >= zeros.first) {
    write_zeros(zeros);
    return;
  }
  __shared__ __align__(16) unsigned keys[kRankTile];
  __shared__ unsigned counts[kRankShares][kRankTokens];
  const int count = (int)p.tokens, mine = threadIdx.x % kRankTokens, share = threadIdx.x / kRankTokens;
  const int first = blockIdx.x * kRankTokens, token = first + mine;
  const unsigned key = token < count ? key_at(p, token) : 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *joins = 0;
  unsigned below = 0;
  unsigned next[kRankTile / kRankThreads];  // the next tile, on its way while this one is compared
  auto load = [&](int tile) {
#pragma unroll
    for (int i = 0; i < kRankTile / kRankThreads; ++i) {
      const int at = tile + i * kRankThreads + threadIdx.x;
      next[i] = at < count ? key_at(p, at) : 0xffffffffu;  // (keys behind the last one are smaller than none)
    }
  };
  load(0);
  for (int tile = 0; tile < count; tile += kRankTile) {
    const int held = min(kRankTile, count - tile);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kRankTile / kRankThreads; ++i) keys[i * kRankThreads + threadIdx.x] = next[i];
    __syncthreads();
    if (tile + kRankTile < count) load(tile + kRankTile);
    // four keys at a time, the shares in turn: those of tokens before this CTA's (equal ones come first), its own, and the rest
    const int own = min(max(first - tile, 0), held), after = min(max(first + kRankTokens - tile, 0), held);
    constexpr int kStep = 4 * kRankShares;
    int i = 4 * share;
#pragma unroll 4
    for (; i < own; i += kStep) {
      const uint4 k = *reinterpret_cast<const uint4*>(keys + i);
      below += (k.x <= key) + (k.y <= key) + (k.z <= key) + (k.w <= key);
    }
    for (; i < after; i += kStep) {
      const uint4 k = *reinterpret_cast<const uint4*>(keys + i);
      const int at = tile + i;
      below += (k.x < key || (k.x == key && at < token)) + (k.y < key || (k.y == key && at + 1 < token)) +
               (k.z < key || (k.z == key && at + 2 < token)) + (k.w < key || (k.w == key && at + 3 < token));
    }
#pragma unroll 4
    for (; i < held; i += kStep) {
      const uint4 k = *reinterpret_cast<const uint4*>(keys + i);
      below += (k.x < key) + (k.y < key) + (k.z < key) + (k.w < key);
    }
  }
  counts[share][mine] = below;
  __syncthreads();
  if (share == 0 && token < count) {
#pragma unroll
    for (int s = 1; s < kRankShares; ++s) below += counts[s][mine];
    sorted[below] = make_uint2(key, token);
  }
}

// More tokens: a least-significant-digit radix sort.  Up to kParts CTAs have a contiguous part of the tokens each; a pass counts
// the digits of each part, finds out where its tokens of each digit begin and puts them there, tile by tile.
constexpr int kParts = 16 * kSMs;
// Every CTA adds up the counts of so few parts by itself.  (The whole gradient, 16 000 tokens: 31 us, with a launch for it 39;
// 250 000: 78, with it 61.)
constexpr int kPartsUnscanned = 64;
constexpr int kTileThreads = kZeroThreads;
constexpr int kTileWarps = kTileThreads / 32;
constexpr int kTileItems = 4;           // tokens of a tile per thread (16: 4 000 000 tokens 338 us, with 4 294; 250 000: 81 and 61)
constexpr int kTile = kTileThreads * kTileItems;
constexpr int kMaxDigit = 8;

struct SortPlan {
  int passes, digit;      // bits
  int scanned;            // whether counts become places in a launch of their own
  int parts;
  long long part;         // tokens, whole tiles
};
SortPlan sort_plan(long long tokens, long long n) {
  SortPlan s;
  int bits = 1;
  while (bits < 32 && (n >> bits) > 0) ++bits;  // keys 0..n
  s.passes = (bits + kMaxDigit - 1) / kMaxDigit;
  s.digit = (bits + s.passes - 1) / s.passes;
  if (s.digit < 2) s.digit = 2;  // (four counts are read at a time)
  const long long tiles = (tokens + kTile - 1) / kTile;
  s.part = (tiles + kParts - 1) / kParts * kTile;
  s.parts = (int)((tokens + s.part - 1) / s.part);
  s.scanned = s.parts > kPartsUnscanned;
  return s;
}

// counts[part * digits + digit].  `pairs`: (key, token) as the pass before left them; the first pass reads the ids.
__global__ void __launch_bounds__(kTileThreads) sort_count_kernel(LookupGradParams p, ZeroPart zeros, SortPlan plan,
                                                                  const uint2* pairs, int shift, unsigned* counts,
                                                                  unsigned* joins) {
  next_launch_may_start();
  wait_for_launch_before();
  if ((int)blockIdx.x >= zeros.first) {
    write_zeros(zeros);
    return;
  }
  const int digits = 1 << plan.digit;
  __shared__ unsigned bins[1 << kMaxDigit];
  for (int i = threadIdx.x; i < digits; i += kTileThreads) bins[i] = 0;
  if (joins && blockIdx.x == 0 && threadIdx.x == 0) *joins = 0;
  __syncthreads();
  const long long begin = blockIdx.x * plan.part, end = min(begin + plan.part, p.tokens);
  for (long long tile = begin; tile < end; tile += kTile) {
    unsigned key[kTileItems];
#pragma unroll
    for (int i = 0; i < kTileItems; ++i) {
      const long long at = tile + i * kTileThreads + threadIdx.x;
      key[i] = at >= end ? 0 : pairs ? pairs[at].x : key_at(p, at);
    }
#pragma unroll
    for (int i = 0; i < kTileItems; ++i) {
      const bool live = tile + i * kTileThreads + threadIdx.x < end;
      const unsigned digit = live ? (key[i] >> shift) & (digits - 1) : 0xffffffffu;
      // one addition for all lanes with the same digit: a frequent token would serialise them
      const unsigned peers = __match_any_sync(FULL, digit);
      if (live && (peers & ((1u << lane_id()) - 1)) == 0) atomicAdd(bins + digit, __popc(peers));
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < digits; i += kTileThreads) counts[blockIdx.x * digits + i] = bins[i];
}

// Exclusive sum of one value per thread over a CTA of kTileThreads.
__device__ __forceinline__ unsigned block_exclusive(unsigned x, unsigned* scratch /* kTileWarps */) {
  const int lane = lane_id(), warp = threadIdx.x >> 5;
  unsigned upto = x;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const unsigned y = __shfl_up_sync(FULL, upto, off);
    if (lane >= off) upto += y;
  }
  if (lane == 31) scratch[warp] = upto;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kTileWarps; ++w) upto += w < warp ? scratch[w] : 0;
  return upto - x;
}

// For each digit, one CTA: counts become the tokens of that digit in the parts before, and totals[digit] their number in all.
constexpr int kScanEach = (kParts + kTileThreads - 1) / kTileThreads;
__global__ void __launch_bounds__(kTileThreads) sort_scan_kernel(unsigned* counts, unsigned* totals, int digits, int parts) {
  __shared__ unsigned scratch[kTileThreads / 32];
  next_launch_may_start();
  wait_for_launch_before();
  const int digit = blockIdx.x;
  unsigned c[kScanEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kScanEach; ++i) {
    const int part = threadIdx.x * kScanEach + i;
    c[i] = part < parts ? counts[part * digits + digit] : 0;
    sum += c[i];
  }
  unsigned before = block_exclusive(sum, scratch);
  if (threadIdx.x == kTileThreads - 1) totals[digit] = before + sum;
#pragma unroll
  for (int i = 0; i < kScanEach; ++i) {
    const int part = threadIdx.x * kScanEach + i;
    if (part < parts) counts[part * digits + digit] = before;
    before += c[i];
  }
}

// Rank of each of a warp's keys (lane l holds items l, 32 + l, ..) among the earlier keys of the warp with the same
// digit; counts[digit] ends as the warp's number of keys with that digit.
__device__ __forceinline__ void warp_ranks(const unsigned (&key)[kTileItems], int shift, unsigned mask, int valid,
                                           unsigned short* counts, unsigned (&rank)[kTileItems]) {
  const unsigned earlier = (1u << lane_id()) - 1;
#pragma unroll
  for (int i = 0; i < kTileItems; ++i) {
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

// Every tile is put in order in shared memory first, so that what goes to one digit's places is written side by side.
__global__ void __launch_bounds__(kTileThreads) sort_place_kernel(LookupGradParams p, ZeroPart zeros, SortPlan plan,
                                                                  const uint2* pairs, int shift, const unsigned* counts,
                                                                  uint2* sorted) {
  next_launch_may_start();
  if ((int)blockIdx.x >= zeros.first) {
    wait_for_launch_before();
    write_zeros(zeros);
    return;
  }
  constexpr int kDigits = 1 << kMaxDigit;
  static_assert(kDigits == kTileThreads, "a digit per thread");
  __shared__ unsigned short warp_counts[kTileWarps * kDigits];
  __shared__ unsigned starts[kDigits], before[kDigits], scratch[2][kTileWarps];
  __shared__ uint2 tile_pairs[kTile];
  const int digits = 1 << plan.digit, warp = threadIdx.x >> 5, lane = lane_id(), parts = plan.parts;
  const long long part_begin = blockIdx.x * plan.part, part_end = min(part_begin + plan.part, p.tokens);
  unsigned key[kTileItems], token[kTileItems], rank[kTileItems];
  auto load = [&](long long tile) {
    const long long begin = tile + warp * 32 * kTileItems + lane;
#pragma unroll
    for (int i = 0; i < kTileItems; ++i) {
      const long long at = begin + i * 32;
      if (at < part_end) {
        const uint2 pair = pairs ? pairs[at] : make_uint2(key_at(p, at), (unsigned)at);
        key[i] = pair.x;
        token[i] = pair.y;
      }
    }
  };
  // tokens of each digit in all parts, and in the ones before this
  if (plan.scanned) {
    wait_for_launch_before();
    load(part_begin);
    if ((int)threadIdx.x < digits) {
      starts[threadIdx.x] = counts[parts * digits + threadIdx.x];
      before[threadIdx.x] = counts[blockIdx.x * digits + threadIdx.x];
    }
  } else {
    // every warp takes some of the parts, a lane four digits
    for (int i = threadIdx.x; i < digits; i += kTileThreads) starts[i] = before[i] = 0;
    wait_for_launch_before();
    load(part_begin);
    __syncthreads();
    for (int d = 4 * lane; d < digits; d += 128) {
      unsigned all[4] = {0, 0, 0, 0}, earlier[4] = {0, 0, 0, 0};
#pragma unroll 8
      for (int i = warp; i < parts; i += kTileWarps) {
        const uint4 c = *reinterpret_cast<const uint4*>(counts + i * digits + d);
        const bool earlier_part = i < (int)blockIdx.x;
        all[0] += c.x, all[1] += c.y, all[2] += c.z, all[3] += c.w;
        earlier[0] += earlier_part ? c.x : 0, earlier[1] += earlier_part ? c.y : 0;
        earlier[2] += earlier_part ? c.z : 0, earlier[3] += earlier_part ? c.w : 0;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        atomicAdd(starts + d + k, all[k]);
        atomicAdd(before + d + k, earlier[k]);
      }
    }
  }
  __syncthreads();
  const bool mine = (int)threadIdx.x < digits;  // the thread's digit, and where its next token goes
  unsigned next = block_exclusive(mine ? starts[threadIdx.x] : 0, scratch[0]) + (mine ? before[threadIdx.x] : 0);
  for (long long tile = part_begin; tile < part_end; tile += kTile) {
    if (tile > part_begin) load(tile);
    for (int i = threadIdx.x; i < kTileWarps * digits / 2; i += kTileThreads) reinterpret_cast<unsigned*>(warp_counts)[i] = 0;
    const int held = (int)min((long long)kTile, part_end - tile);
    const int valid = max(0, min(32 * kTileItems, held - warp * 32 * kTileItems));
    __syncthreads();
    warp_ranks(key, shift, digits - 1, valid, warp_counts + warp * digits, rank);
    __syncthreads();
    // a digit's tokens in the warps before, and in the tile
    unsigned total = 0;
    if (mine) {
#pragma unroll
      for (int w = 0; w < kTileWarps; ++w) {
        const unsigned c = warp_counts[w * digits + threadIdx.x];
        warp_counts[w * digits + threadIdx.x] = (unsigned short)total;
        total += c;
      }
    }
    const unsigned local = block_exclusive(total, scratch[1]);
    if (mine) {
      starts[threadIdx.x] = local;         // the digit's first place in the tile
      before[threadIdx.x] = next - local;  // from a place in the tile to one in the result
      next += total;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTileItems; ++i) {
      if (i * 32 + lane < valid) {
        const unsigned digit = (key[i] >> shift) & (digits - 1);
        tile_pairs[starts[digit] + warp_counts[warp * digits + digit] + rank[i]] = make_uint2(key[i], token[i]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTileItems; ++i) {
      const int at = i * kTileThreads + threadIdx.x;
      if (at < held) {
        const uint2 pair = tile_pairs[at];
        sorted[before[(pair.x >> shift) & (digits - 1)] + at] = pair;
      }
    }
    __syncthreads();
  }
}

// ---- gradient: sums over the sorted tokens --------------------------------------------------------------------------

// The sorted tokens are cut into chunks of equal length, whatever rows they belong to: a frequent token makes no CTA's work
// longer.  A row whose tokens all lie in one chunk is written there; of a row that crosses a border each chunk leaves a
// partial sum in fp32 (heads: of the row that the chunk before began; tails: of the row that goes on in the next one), and
// join_kernel adds those up.
constexpr int kSumThreads = 256;
constexpr int kInFlight = 4;
constexpr int kMostChunk = 64;
constexpr int kSumLanes = 8;   // threads of a chunk at least

struct SumPlan {
  int chunk;         // tokens, a multiple of 2 * kInFlight
  long long chunks;
};
SumPlan sum_plan(long long tokens, long long d) {
  SumPlan s;
  // Chunks of 64 tokens where that leaves every SM some 14 000 values to add side by side, and of many tokens; shorter ones for
  // fewer tokens, but the shorter they are the more partial sums there are to join.  (At least 16 instead: 166 845 tokens of 123
  // dimensions 86 us, now 76; 65 536 of 768 101 and 90.  At least 8 instead of 16: 6457 of 954 dimensions 41 us, now 37.)
  s.chunk = kMostChunk;
  const int least = tokens > 32768 ? 64 : tokens > 8192 ? 32 : tokens > 2048 ? 16 : 8;
  while (s.chunk > least && tokens / s.chunk * d < (long long)kSMs * 14'000) s.chunk /= 2;
  s.chunks = (tokens + s.chunk - 1) / s.chunk;
  return s;
}

template <class O, int N>
__device__ __forceinline__ void write_row(const LookupGradParams& p, unsigned row, long long c, const float (&sum)[N]) {
  O* at = static_cast<O*>(p.out) + (long long)row * p.d + c;
  O v[N];
  if (p.accumulate) {
    load_many<O, N>(at, v);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = from_f32<O>(to_f32(v[i]) + sum[i] * p.scale);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = from_f32<O>(sum[i] * p.scale);
  }
  store_many<O, N>(at, v);
}

// `lanes` threads have a chunk (of up to lanes * N dimensions); kInFlight rows of the gradient are on their way to each.  A
// thread has N neighbouring values or, of rows that are no whole words (kApart), N values `lanes` apart.  Bound: HBM latency of
// rows anywhere (1 000 003 of 50 floats in 100 us, 3.8 TB/s; eight rows on their way instead of four: the same).
template <class G, class O, int N, bool kApart>
__global__ void __launch_bounds__(kSumThreads, kApart || sizeof(G) * N > 8 ? 3 : 4)
  sum_kernel(LookupGradParams p, SumPlan plan, const uint2* sorted, float* heads, float* tails, unsigned* joins,
             unsigned* join_list, int lanes) {
  const int group = threadIdx.x / lanes, lane = threadIdx.x % lanes, groups = blockDim.x / lanes;
  const long long chunk = (long long)blockIdx.x * groups + group;
  next_launch_may_start();
  wait_for_launch_before();
  __shared__ __align__(16) unsigned chunk_keys[kSumThreads / kSumLanes][kMostChunk];
  __shared__ __align__(16) unsigned chunk_tokens[kSumThreads / kSumLanes][kMostChunk];
  const unsigned none = (unsigned)p.n;
  const long long begin = chunk * plan.chunk, end = min(begin + plan.chunk, p.tokens);
  for (int i = lane; i < plan.chunk; i += lanes) {  // (the end of the last chunk as empty slots)
    const uint2 pair = begin + i < end ? sorted[begin + i] : make_uint2(none, 0);
    chunk_keys[group][i] = pair.x;
    chunk_tokens[group][i] = pair.y;
  }
  __syncthreads();
  if (chunk >= plan.chunks) return;
  const long long c = (long long)blockIdx.y * lanes * N + (kApart ? lane : lane * N);
  if (c >= p.d) return;
  const int held = kApart ? (int)min((long long)N, (p.d - c + lanes - 1) / lanes) : N;  // values
  const G* grad = static_cast<const G*>(p.grad) + c;
  const unsigned before = begin > 0 ? sorted[begin - 1].x : none, after = end < p.tokens ? sorted[end].x : none;
  unsigned row = chunk_keys[group][0];
  bool head = row == before;  // the row that the chunk begins with is another chunk's as well
  float sum[N];
#pragma unroll
  for (int i = 0; i < N; ++i) sum[i] = 0.0f;
  auto partial = [&](float* to) {
    to += chunk * p.d + c;
    if constexpr (kApart) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < held) to[j * lanes] = sum[j];
    } else {
      store_many<float, N>(to, sum);
    }
  };
  auto write = [&] {
    if constexpr (kApart) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float one[1] = {sum[j]};
        if (j < held) write_row<O, 1>(p, row, c + j * lanes, one);
      }
    } else {
      write_row<O, N>(p, row, c, sum);
    }
  };
  // (whole words: a value of 16 bits that waits by itself takes a register)
  using Word = typename WordOf<kApart ? sizeof(G) : sizeof(G) * N>::type;
  constexpr int kWords = kApart ? N : 1;
  auto fetch = [&](int t, Word (&word)[kInFlight][kWords]) {
    const uint4 k = *reinterpret_cast<const uint4*>(chunk_keys[group] + t);
    const uint4 at = *reinterpret_cast<const uint4*>(chunk_tokens[group] + t);
    const unsigned key[kInFlight] = {k.x, k.y, k.z, k.w}, token[kInFlight] = {at.x, at.y, at.z, at.w};
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      if (key[i] == none) continue;
      const G* from = grad + (long long)token[i] * p.grad_stride;
#pragma unroll
      for (int j = 0; j < kWords; ++j)
        if (!kApart || j < held) word[i][j] = __ldcs(reinterpret_cast<const Word*>(from + (kApart ? j * lanes : 0)));
    }
  };
  auto add = [&](int t, const Word (&word)[kInFlight][kWords]) {
    const uint4 k = *reinterpret_cast<const uint4*>(chunk_keys[group] + t);
    const unsigned key[kInFlight] = {k.x, k.y, k.z, k.w};
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      if (key[i] != row) {
        if (key[i] == none) return;  // nothing but empty slots from here on, or the end
        if (head)
          partial(heads);
        else
          write();
        head = false;
        row = key[i];
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] = 0.0f;
      }
      if constexpr (kApart) {
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] += to_f32(*reinterpret_cast<const G*>(&word[i][j]));
      } else {
        const Vec<G, N> v = *reinterpret_cast<const Vec<G, N>*>(&word[i][0]);
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] += to_f32(v.v[j]);
      }
    }
  };
  if (row == none) return;  // a chunk of empty slots
  // two sets of words in turn: one on its way while the other one is added
  Word even[kInFlight][kWords], odd[kInFlight][kWords];
  fetch(0, even);
  for (int t = 0; t < plan.chunk; t += 2 * kInFlight) {
    fetch(t + kInFlight, odd);
    add(t, even);
    if (t + 2 * kInFlight < plan.chunk) fetch(t + 2 * kInFlight, even);
    add(t + kInFlight, odd);
  }
  if (head) {
    partial(heads);
  } else if (row == after) {
    partial(tails);
    if (c == 0) join_list[atomicAdd(joins, 1u)] = (unsigned)chunk;
  } else {
    write();
  }
}

// Rows that cross borders of chunks.  A warp takes one of them and 32 * kEach dimensions; of a row with many partial sums the
// CTA's warps add up a share each.  Bound: latency, some eight dependent loads (8 to 18 us).  Of up to 32 dimensions 32 partial
// sums are on their way at a time: 300 000 tokens of 17 dimensions, half of them of a few rows, 68 us with kEach 1, 81 with 4.
constexpr int kJoinWarps = 8;
constexpr int kJoinBlocks = 48 / kJoinWarps * kSMs;
constexpr int kJoinLoads = 32;       // in flight per lane
constexpr long long kJoinAlone = 20;  // partial sums that a warp adds up by itself

template <class O, int kEach>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(LookupGradParams p, SumPlan plan, const uint2* sorted,
                                                               const float* heads, const float* tails,
                                                               const unsigned* joins, const unsigned* join_list) {
  constexpr int kJoinDims = 32 * kEach;
  __shared__ float sums[kJoinWarps][kJoinDims];
  __shared__ long long first_of[kJoinWarps], parts_of[kJoinWarps];
  __shared__ unsigned row_of[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = lane_id();
  wait_for_launch_before();
  const long long count = *joins, items = count * ((p.d + kJoinDims - 1) / kJoinDims);
  for (long long base = (long long)blockIdx.x * kJoinWarps; base < items; base += (long long)gridDim.x * kJoinWarps) {
    const long long item = base + warp;
    long long chunk = 0, parts = 0;
    unsigned row = 0;
    if (item < items) {
      chunk = join_list[item % count];  // (a CTA's warps take different rows: the longest ones are not all its own)
      row = sorted[(chunk + 1) * plan.chunk].x;
      // the last chunk that begins with the row: 32 candidates at a time, the next ones first
      long long low = chunk + 1, step = 1;
      for (;;) {
        const long long at = low + (lane + 1) * step;
        const unsigned same = __ballot_sync(FULL, at < plan.chunks && sorted[min(at, plan.chunks - 1) * plan.chunk].x == row);
        const int reached = __popc(same);  // they are the first ones
        low += reached * step;
        if (reached == 32) {
          step *= 32;
        } else if (step == 1) {
          break;
        } else {
          step /= 32;
        }
      }
      parts = low - chunk + 1;  // one tail, the rest heads
    }
    auto add = [&](long long from_chunk, long long from, long long to, long long column, float (&sum)[kEach]) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) sum[i] = 0.0f;
      if (from == 0 && to > 0) {
        const float* tail = tails + from_chunk * p.d + column * kJoinDims + lane;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
          if (column * kJoinDims + lane + 32 * i < p.d) sum[i] = tail[32 * i];
        ++from;
      }
      const float* head = heads + (from_chunk + from) * p.d + column * kJoinDims + lane;
#pragma unroll(kJoinLoads / kEach)
      for (long long k = from; k < to; ++k, head += p.d) {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
          if (column * kJoinDims + lane + 32 * i < p.d) sum[i] += head[32 * i];
      }
    };
    auto write = [&](unsigned to_row, long long column, const float (&sum)[kEach]) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const long long c = column * kJoinDims + lane + 32 * i;
        const float one[1] = {sum[i]};
        if (c < p.d) write_row<O, 1>(p, to_row, c, one);
      }
    };
    if (item < items && parts <= kJoinAlone) {
      float sum[kEach];
      add(chunk, 0, parts, item / count, sum);
      write(row, item / count, sum);
    }
    if (lane == 0) {
      first_of[warp] = chunk;
      parts_of[warp] = parts;
      row_of[warp] = row;
    }
    __syncthreads();
    for (int w = 0; w < kJoinWarps; ++w) {
      if (parts_of[w] <= kJoinAlone) continue;
      const long long share = (parts_of[w] + kJoinWarps - 1) / kJoinWarps, column = (base + w) / count;
      float sum[kEach];
      add(first_of[w], warp * share, min(parts_of[w], (warp + 1) * share), column, sum);
#pragma unroll
      for (int i = 0; i < kEach; ++i) sums[warp][lane + 32 * i] = sum[i];
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          sum[i] = sums[0][lane + 32 * i];
#pragma unroll
          for (int v = 1; v < kJoinWarps; ++v) sum[i] += sums[v][lane + 32 * i];
        }
        write(row_of[w], column, sum);
      }
      __syncthreads();
    }
    __syncthreads();
  }
}

// ---- gradient: few tokens -------------------------------------------------------------------------------------------

// Few tokens: one launch without a sort of all.  A CTA has kFewBytes of the result: it writes zeros, looks for its
// rows among all ids, puts their tokens in order and writes the sums over the zeros.  Bound: latency.
constexpr int kFewTokens = 512;
constexpr int kFewBytes = 16 * 1024;
constexpr int kFewThreads = 256;
constexpr int kFewAlone = 16;  // tokens of a row that one group of lanes adds up by itself
constexpr int kFewLoads = 8;   // in flight per thread

// Where that is better: rows short enough for a CTA to add up the most frequent one, and very few tokens, or ones that find many CTAs
// and zeros that do not take longer than the sort would.  (Caches cold.  128 tokens: 1000 rows of 8 floats 10 us, sorted 15; 32 000 of
// 256 13 and 17; 524 288 of 256 78 and 83; one row of 4096 bytes of 16 000 35 and 24.  511 tokens: 1000 rows of 8 29 and 15; 8000 of 256 12
// and 17; 32 000 16 and 17; 524 288 96 and 85.  It loses where many tokens are of rows next to each other: 511 of 32 000 rows
// with the frequent ones in front 25 and 17.)
constexpr int kFewAnywhere = 128;  // tokens
bool few(const LookupGradParams& p, long long row_bytes) {
  const long long bytes = p.n * row_bytes;
  return !p.accumulate && row_bytes <= 2048 &&
         (p.tokens <= kFewAnywhere ||
          (p.tokens <= kFewTokens && bytes <= (64 << 20) && bytes >= (long long)kSMs * kFewBytes));
}

template <class G, class O, int N>
__global__ void __launch_bounds__(kFewThreads) few_kernel(LookupGradParams p, int rows_each, int lanes) {
  __shared__ unsigned masks[kFewTokens / 32];
  __shared__ unsigned short row_of[kFewTokens], list_row[kFewTokens], list_token[kFewTokens];
  __shared__ unsigned short sorted_row[kFewTokens], sorted_token[kFewTokens], long_rows[kFewTokens / kFewAlone];
  __shared__ int long_count;
  __shared__ __align__(16) float partial[kFewThreads * N];
  next_launch_may_start();
  wait_for_launch_before();
  const long long row0 = (long long)blockIdx.x * rows_each;
  const int rows = (int)min((long long)rows_each, p.n - row0), d = (int)p.d, tokens = (int)p.tokens;
  {
    unsigned char* to = static_cast<unsigned char*>(p.out) + row0 * d * sizeof(O);
    const int bytes = rows * d * (int)sizeof(O), head = min(bytes, (int)(-reinterpret_cast<uintptr_t>(to) & 15));
    const int words = (bytes - head) / 16, tail = (bytes - head) % 16;
    for (int i = threadIdx.x; i < words; i += kFewThreads) reinterpret_cast<uint4*>(to + head)[i] = make_uint4(0, 0, 0, 0);
    if ((int)threadIdx.x < head) to[threadIdx.x] = 0;
    if ((int)threadIdx.x < tail) to[head + 16 * words + threadIdx.x] = 0;
  }
  bool any = false;
  if (threadIdx.x == 0) long_count = 0;
  for (int base = 0; base < tokens; base += kFewThreads) {
    const int t = base + threadIdx.x;
    const long long id = t < tokens ? id_at(p.ids, p.ids64, t) : -1;
    const bool mine = id >= row0 && id < row0 + rows;
    const unsigned mask = __ballot_sync(FULL, mine);
    if (lane_id() == 0) masks[t / 32] = mask;
    if (mine) row_of[t] = (unsigned short)(id - row0);
    any = any || mine;
  }
  if (!__syncthreads_or(any)) return;
  // the tokens of its rows in their order, then by row
  int count = 0;
  for (int base = 0; base < tokens; base += kFewThreads) {
    const int t = base + threadIdx.x, word = t / 32;
    int before = count;
    for (int w = base / 32; w < word; ++w) before += __popc(masks[w]);
    if (masks[word] >> (t & 31) & 1) {
      const int at = before + __popc(masks[word] & ((1u << (t & 31)) - 1));
      list_row[at] = row_of[t];
      list_token[at] = (unsigned short)t;
    }
    for (int w = base / 32; w < (base + kFewThreads) / 32; ++w) count += __popc(masks[w]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kFewThreads) {
    const int row = list_row[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < count; ++j) rank += list_row[j] < row || (list_row[j] == row && j < i);
    sorted_row[rank] = (unsigned short)row;
    sorted_token[rank] = list_token[i];
  }
  __syncthreads();
  const int group = threadIdx.x / lanes, lane = threadIdx.x % lanes, groups = kFewThreads / lanes;
  const G* grad = static_cast<const G*>(p.grad);
  auto sum_of = [&](int from, int to, int c, float (&sum)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = 0.0f;
    for (int k = from; k < to; k += kFewLoads) {
      Vec<G, N> v[kFewLoads];
#pragma unroll
      for (int u = 0; u < kFewLoads; ++u)
        if (k + u < to) v[u] = load_vec<G, N>(grad + (long long)sorted_token[k + u] * p.grad_stride + c);
#pragma unroll
      for (int u = 0; u < kFewLoads; ++u) {
        if (k + u >= to) break;
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] += to_f32(v[u].v[j]);
      }
    }
  };
  for (int s = group; s < count; s += groups) {
    const int row = sorted_row[s];
    if (s > 0 && sorted_row[s - 1] == row) continue;
    if (s + kFewAlone < count && sorted_row[s + kFewAlone] == row) {
      if (lane == 0) long_rows[atomicAdd(&long_count, 1)] = (unsigned short)s;
      continue;
    }
    int end = s + 1;
    while (end < count && sorted_row[end] == row) ++end;
    for (int c = lane * N; c < d; c += lanes * N) {
      float sum[N];
      sum_of(s, end, c, sum);
      write_row<O, N>(p, (unsigned)(row0 + row), c, sum);
    }
  }
  __syncthreads();
  // rows of more tokens: a share for each group
  for (int i = 0; i < long_count; ++i) {
    const int s = long_rows[i], row = sorted_row[s];
    int length = 0;
    for (int base = s; base < count; base += kFewThreads)
      length += __syncthreads_count(base + (int)threadIdx.x < count &&
                                    sorted_row[min(base + (int)threadIdx.x, count - 1)] == row);
    const int share = (length + groups - 1) / groups, from = min(length, group * share), to = min(length, from + share);
    for (int base = 0; base < d; base += lanes * N) {
      const int c = base + lane * N;
      float sum[N];
      if (c < d) {
        sum_of(s + from, s + to, c, sum);
        store_many<float, N>(partial + threadIdx.x * N, sum);
      }
      __syncthreads();
      if (group == 0 && c < d) {
        for (int other = 1; other < groups; ++other) {
#pragma unroll
          for (int j = 0; j < N; ++j) sum[j] += partial[(other * lanes + lane) * N + j];
        }
        write_row<O, N>(p, (unsigned)(row0 + row), c, sum);
      }
      __syncthreads();
    }
  }
}

template <class G, class O, int N>
cudaError_t few_t(const LookupGradParams& p, cudaStream_t stream) {
  const int row = (int)(p.d * sizeof(O)), each = kFewBytes / row;
  const long long blocks = (p.n + each - 1) / each;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  return launch_early(few_kernel<G, O, N>, dim3((unsigned)blocks), kFewThreads, 0, stream, p, each,
                      next_pow2((p.d + N - 1) / N, kFewThreads));
}

struct GradSpace {
  uint2* pairs[2];  // (key, token)
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
  const SortPlan plan = sort_plan(tokens, n);
  const bool ranked = tokens <= kRankMost;
  for (int i = 0; i < 2; ++i) s.pairs[i] = reinterpret_cast<uint2*>(take(ranked && i ? 0 : 2 * tokens));
  s.counts = reinterpret_cast<unsigned*>(take(ranked ? 0 : (long long)(plan.parts + 1) << plan.digit));
  s.joins = reinterpret_cast<unsigned*>(take(1));
  s.join_list = reinterpret_cast<unsigned*>(take(sums.chunks));
  s.heads = reinterpret_cast<float*>(take(sums.chunks * d));
  s.tails = reinterpret_cast<float*>(take(sums.chunks * d));
  s.bytes = used;
  return s;
}

template <class G, class O, int N, bool kApart>
cudaError_t sum_t(const LookupGradParams& p, const SumPlan& plan, const GradSpace& s, int at, cudaStream_t stream) {
  // more than a warp: as many warps as it takes, in columns of equal width
  const long long need = (p.d + N - 1) / N, columns = (need + kSumThreads - 1) / kSumThreads;
  int lanes = need > 32 ? (int)((need + columns - 1) / columns + 31) / 32 * 32 : next_pow2(need, 32);
  if (lanes < kSumLanes) lanes = kSumLanes;
  const int groups = kSumThreads / lanes;
  const long long blocks = (plan.chunks + groups - 1) / groups;
  if (blocks > 0x7fffffffll || columns > 65535) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)blocks, (unsigned)columns);
  return launch_early(sum_kernel<G, O, N, kApart>, grid, lanes * groups, 0, stream, p, plan, s.pairs[at], s.heads,
                      s.tails, s.joins, s.join_list, lanes);
}

template <class G, class O>
cudaError_t grad_t(const LookupGradParams& p, cudaStream_t stream) {
  const int w = word_bytes(reinterpret_cast<uintptr_t>(p.grad) | (unsigned long long)(p.grad_stride * sizeof(G)) |
                           (unsigned long long)(p.d * sizeof(G)));
  const int to = word_bytes(reinterpret_cast<uintptr_t>(p.out)) / (int)sizeof(O) * (int)sizeof(G);
  if (few(p, p.d * (long long)sizeof(O))) {
    if (w == 16 && to * sizeof(O) >= 16 * sizeof(G)) return few_t<G, O, 16 / sizeof(G)>(p, stream);
    if (w >= 8 && to >= 8) return few_t<G, O, 8 / sizeof(G)>(p, stream);
    if (w >= 4 && to >= 4) return few_t<G, O, 4 / sizeof(G)>(p, stream);
    return few_t<G, O, 1>(p, stream);
  }
  const SumPlan plan = sum_plan(p.tokens, p.d);
  const GradSpace s = grad_space(p.tokens, p.n, p.d, p.workspace);
  // the zeros in equal parts with each of the sort's launches, by four CTAs per SM
  const unsigned long long bytes = p.accumulate ? 0 : (unsigned long long)p.n * p.d * sizeof(O);
  const unsigned long long words = (bytes - (bytes < 16 ? bytes : -reinterpret_cast<uintptr_t>(p.out) & 15)) / 16;
  auto zeros = [&](int first, int launch, int launches) {
    ZeroPart z;
    z.first = first;
    z.begin = words / launches * launch;
    z.words = launch + 1 == launches ? words - z.begin : words / launches;
    z.out = static_cast<unsigned char*>(p.out);
    z.bytes = bytes;
    return z;
  };
  // (a CTA is there for the single bytes even if there are no words)
  auto zero_blocks = [&](const ZeroPart& z) { return bytes == 0 ? 0 : z.words / kZeroWords + 1; };
  cudaError_t e;
  int at = 0;
  if (p.tokens <= kRankMost) {
    const ZeroPart z = zeros((int)((p.tokens + kRankTokens - 1) / kRankTokens), 0, 1);
    e = launch_early(sort_rank_kernel, dim3((unsigned)(z.first + zero_blocks(z))), kRankThreads, 0, stream, p, z, s.pairs[0],
                     s.joins);
    if (e != cudaSuccess) return e;
  } else {
    const SortPlan sort = sort_plan(p.tokens, p.n);
    for (int pass = 0; pass < sort.passes; ++pass) {
      const uint2* pairs = pass ? s.pairs[at] : nullptr;
      const int to = pass ? 1 - at : 0, shift = pass * sort.digit;
      const ZeroPart first = zeros(sort.parts, 2 * pass, 2 * sort.passes);
      const ZeroPart second = zeros(sort.parts, 2 * pass + 1, 2 * sort.passes);
      unsigned* joins = pass ? nullptr : s.joins;
      const dim3 grid((unsigned)(first.first + zero_blocks(first)));
      e = launch_early(sort_count_kernel, grid, kTileThreads, 0, stream, p, first, sort, pairs, shift, s.counts, joins);
      if (e != cudaSuccess) return e;
      if (sort.scanned) {
        unsigned* totals = s.counts + ((size_t)sort.parts << sort.digit);
        e = launch_early(sort_scan_kernel, dim3(1u << sort.digit), kTileThreads, 0, stream, s.counts, totals, 1 << sort.digit,
                         sort.parts);
        if (e != cudaSuccess) return e;
      }
      e = launch_early(sort_place_kernel, dim3((unsigned)(second.first + zero_blocks(second))), kTileThreads, 0, stream, p, second,
                       sort, pairs, shift, s.counts, s.pairs[to]);
      if (e != cudaSuccess) return e;
      at = to;
    }
  }
  if (w == 16 && to * sizeof(O) >= 16 * sizeof(G))
    e = sum_t<G, O, 16 / sizeof(G), false>(p, plan, s, at, stream);
  else if (w >= 8 && to >= 8)
    e = sum_t<G, O, 8 / sizeof(G), false>(p, plan, s, at, stream);
  else if (w >= 4 && to >= 4 && (sizeof(G) == 2 || p.d <= kSumThreads))
    // (whole words of one float, of rows that a CTA has threads for: 60 000 tokens of 17 floats 42 us, 55 with floats apart;
    // 20 000 of 953: 79 and 75)
    e = sum_t<G, O, 4 / sizeof(G), false>(p, plan, s, at, stream);
  else
    e = sum_t<G, O, 4, true>(p, plan, s, at, stream);
  if (e != cudaSuccess || plan.chunks < 2) return e;
  auto join = [&](auto* kernel, int dims) {
    const long long items = plan.chunks * ((p.d + dims - 1) / dims), wanted = (items + kJoinWarps - 1) / kJoinWarps;
    return launch_early(kernel, dim3((unsigned)(wanted < kJoinBlocks ? wanted : kJoinBlocks)), kJoinWarps * 32, 0, stream, p,
                        plan, s.pairs[at], s.heads, s.tails, s.joins, s.join_list);
  };
  return p.d <= 32 ? join(join_kernel<O, 1>, 32) : join(join_kernel<O, 4>, 128);
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
