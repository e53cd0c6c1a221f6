// Rows of a table in 4 bits: packing, unpacking, and products of queries with all rows.
//
// A value is (code - 8) * scale: a code of 0..15 per value and a bfloat16 scale per `group` consecutive dimensions of a row.
// A row's codes are 32-bit words of eight values (16 bytes per block of 32 dimensions, the last one filled up with code 8).
// Blocks lie in fours (the last of a row as many as are left, m): word t*m + j of a four holds dimensions 8t..8t+7 of its
// block j, the even ones in nibbles 0..3, the odd ones in nibbles 4..7.  So a lane's 16 bytes of a row are its part of four
// steps of the matrix instruction over 32 dimensions each, a group of 32 or 64 dimensions ends between two steps, and
// w & 0x000f000f is a pair of consecutive values in two halves of a register.
#include "scores4.cuh"

#include <type_traits>

namespace hnsw {

namespace {

// Byte offset in a row of the word that holds dimensions 8 * index .. 8 * index + 7
__device__ __forceinline__ int word_offset(int index, int blocks) {
  const int four = index >> 4, block = (index >> 2) & 3, t = index & 3;
  return 64 * four + 4 * (t * min(4, blocks - 4 * four) + block);
}

// ---- packing --------------------------------------------------------------------------------------------------------

constexpr int kPackThreads = 256;

// (d is a multiple of N)
template <class T, int N>
__device__ __forceinline__ void load_eight(const T* row, int dim, int d, T (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += N) {
    T w[N];
#pragma unroll
    for (int j = 0; j < N; ++j) w[j] = from_f32<T>(0.0f);
    if (dim + i < d) load_many<T, N>(row + dim + i, w);
#pragma unroll
    for (int j = 0; j < N; ++j) v[i + j] = w[j];
  }
}

// The larger one; NaN if one of them is.
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// (A NaN becomes its group's scale, and so NaN all that the group's codes stand for: they have no room for one.)
template <class T>
__device__ __forceinline__ float largest(const T (&v)[8], float most) {
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max_or_nan(most, fabsf(to_f32(v[i])));
  return most;
}

__device__ __forceinline__ __nv_bfloat16 scale_of(float most) { return __float2bfloat16_rn(__fmul_rn(most, 1.0f / 7.0f)); }

__device__ __forceinline__ constexpr int nibble_shift(int i) { return 4 * ((i >> 1) + 4 * (i & 1)); }

__device__ __forceinline__ bool ordinary(float step) { return step > 1e-30f && step < 1e30f; }  // so is its reciprocal

// The codes of eight values.  step: an ordinary scale.
template <class T>
__device__ __forceinline__ unsigned codes_of(const T (&v)[8], float step) {
  // Added to a small number, this leaves its nearest whole number (the even one of two) in the last bits; what else it leaves is
  // taken away for all eight at once.
  constexpr float kWhole = 12582912.0f;
  constexpr unsigned kLess = 0x4b400000u - 8;
  unsigned word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) word -= kLess << nibble_shift(i);
  const float inverse = __frcp_rn(step);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = to_f32(v[i]);
    // The quotient, correctly rounded (16-bit values are halfway between two codes often enough): with a correctly rounded
    // reciprocal one correction by the exact remainder does it (Markstein, Computation of elementary functions on the IBM RISC
    // System/6000 processor, 1990).  Its magnitude is below 7.1, as the scale is the largest value's.
    const float near = x * inverse;
    const float quotient = __fmaf_rn(__fmaf_rn(-near, step, x), inverse, near);
    word += __float_as_uint(quotient + kWhole) << nibble_shift(i);
  }
  return word;
}

// The same with no scale, or with one whose reciprocal is no ordinary number.  (Beside an infinite scale infinities keep their sign, 7
// or -8 times the scale, and 0 times it is a NaN: what was finite is lost.)
template <class T>
__device__ __forceinline__ unsigned codes_of_any(const T (&v)[8], float step) {
  unsigned word = 0;
  for (int i = 0; i < 8; ++i) {
    const float x = to_f32(v[i]);
    const float q = !(step > 0.0f) ? 0.0f : isinf(x) ? x : rintf(__fdiv_rn(x, step));
    word |= (unsigned)((int)fminf(fmaxf(q, -8.0f), 7.0f) + 8) << nibble_shift(i);
  }
  return word;
}

// `lanes` lanes (a power of two, at most a warp) take the words of eight dimensions of kAt rows at once.  Bound: instructions, some
// 20 per value (1 183 514 rows of 50 floats in 60 us, 4.7 TB/s).
template <class T, int N, int kAt>
__global__ void __launch_bounds__(kPackThreads, 4) pack_kernel(const T* rows, long long row_stride, long long n, int d,
                                                               int group_shift, int groups, unsigned char* codes,
                                                               __nv_bfloat16* scales, int lanes) {
  next_launch_may_start();
  wait_for_launch_before();
  const int lane = threadIdx.x & (lanes - 1);
  const int blocks = (d + kBlock - 1) / kBlock, words = 4 * blocks, span = min(lanes, 1 << group_shift);
  const long long row = ((long long)blockIdx.x * (kPackThreads / lanes) + threadIdx.x / lanes) * kAt;
  const T* src = rows + row * row_stride;
  unsigned char* dst = codes + row * (16ll * blocks);
  __nv_bfloat16* to_scales = scales + row * groups;
  T v[kAt][8];
#pragma unroll
  for (int k = 0; k < kAt; ++k) {
    if (row + k < n && 8 * lane < d) {
      load_eight<T, N>(src + k * row_stride, 8 * lane, d, v[k]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = from_f32<T>(0.0f);
    }
  }
  float most[kAt];
#pragma unroll
  for (int k = 0; k < kAt; ++k) most[k] = largest(v[k], 0.0f);
  for (int off = 1; off < span; off <<= 1) {
#pragma unroll
    for (int k = 0; k < kAt; ++k) most[k] = max_or_nan(most[k], __shfl_xor_sync(FULL, most[k], off));
  }
  unsigned word[kAt];
  bool live[kAt], other = false;
#pragma unroll
  for (int k = 0; k < kAt; ++k) {
    most[k] = __bfloat162float(scale_of(most[k]));
    word[k] = codes_of(v[k], most[k]);
    live[k] = row + k < n && lane < words;
    other = other || (live[k] && !ordinary(most[k]));
  }
  if (other) {
#pragma unroll
    for (int k = 0; k < kAt; ++k)
      if (live[k] && !ordinary(most[k])) word[k] = codes_of_any(v[k], most[k]);
  }
  const int g = lane >> group_shift;
#pragma unroll
  for (int k = 0; k < kAt; ++k) {
    if (live[k]) {
      *reinterpret_cast<unsigned*>(dst + k * (16ll * blocks) + word_offset(lane, blocks)) = word[k];
      if (g << group_shift == lane && g < groups) to_scales[k * groups + g] = __float2bfloat16_rn(most[k]);
    }
  }
}

// Rows of more than 32 words: a warp has a row, and 4 x 32 words of it at a time, whole ones without a question (50 000 rows of 2048
// bfloat16 in 58 us, 4.2 TB/s; as it was at 66, with a question at each word 80).  Bound: instructions, issue slots 0.76 in use.
template <class T, int N>
__global__ void __launch_bounds__(kPackThreads) pack_long_kernel(const T* rows, long long row_stride, long long n, int d,
                                                                 int group_shift, int groups, unsigned char* codes,
                                                                 __nv_bfloat16* scales) {
  constexpr int kAt = 4;
  next_launch_may_start();
  wait_for_launch_before();
  const int lane = lane_id();
  const long long row = (long long)blockIdx.x * (kPackThreads / 32) + (threadIdx.x >> 5);
  if (row >= n) return;
  const int blocks = (d + kBlock - 1) / kBlock, words = 4 * blocks, span = 1 << group_shift;
  const T* src = rows + row * row_stride + 8 * lane;
  unsigned char* dst = codes + row * (16ll * blocks);
  __nv_bfloat16* to_scales = scales + row * groups;
  // where a lane's word is among 32 of whole fours, and whether it is the first of its group
  const int at_lane = 64 * (lane >> 4) + 16 * (lane & 3) + 4 * ((lane >> 2) & 3);
  const bool leads = (lane & (span - 1)) == 0;
  auto pass = [&](int begin, auto all_whole) {
    constexpr bool kWhole = decltype(all_whole)::value;
    T v[kAt][8];
    bool whole[kAt];  // 32 whole words, of whole fours
#pragma unroll
    for (int k = 0; k < kAt; ++k) {
      const int first = begin + 32 * k;
      whole[k] = kWhole || 8 * (first + 32) <= d;
      if (whole[k]) {
#pragma unroll
        for (int i = 0; i < 8; i += N) {
          T part[N];
          load_many<T, N>(src + 8 * first + i, part);
#pragma unroll
          for (int j = 0; j < N; ++j) v[k][i + j] = part[j];
        }
      } else {
        load_eight<T, N>(src + 8 * first, 0, d - 8 * (first + lane), v[k]);
      }
    }
    float most[kAt];
#pragma unroll
    for (int k = 0; k < kAt; ++k) most[k] = largest(v[k], 0.0f);
    for (int off = 1; off < span; off <<= 1) {
#pragma unroll
      for (int k = 0; k < kAt; ++k) most[k] = max_or_nan(most[k], __shfl_xor_sync(FULL, most[k], off));
    }
    unsigned word[kAt];
    bool other = false;
#pragma unroll
    for (int k = 0; k < kAt; ++k) {
      if (!kWhole && begin + 32 * k >= words) continue;  // (behind the row, for the whole warp)
      most[k] = __bfloat162float(scale_of(most[k]));
      word[k] = codes_of(v[k], most[k]);
      other = other || ((kWhole || begin + 32 * k + lane < words) && !ordinary(most[k]));
    }
    if (other) {
#pragma unroll
      for (int k = 0; k < kAt; ++k)
        if (!ordinary(most[k])) word[k] = codes_of_any(v[k], most[k]);
    }
#pragma unroll
    for (int k = 0; k < kAt; ++k) {
      const int w = begin + 32 * k + lane;
      if (whole[k]) {
        *reinterpret_cast<unsigned*>(dst + at_lane + 4 * (begin + 32 * k)) = word[k];
        if (leads) to_scales[w >> group_shift] = __float2bfloat16_rn(most[k]);
      } else if (w < words) {
        *reinterpret_cast<unsigned*>(dst + word_offset(w, blocks)) = word[k];
        if (leads && w >> group_shift < groups) to_scales[w >> group_shift] = __float2bfloat16_rn(most[k]);
      }
    }
  };
  int begin = 0;
  for (; 8 * (begin + 32 * kAt) <= d; begin += 32 * kAt) pass(begin, std::true_type());
  if (begin < words) pass(begin, std::false_type());
}

// Groups that are more than a warp's words: a warp per row, every group read twice.
template <class T, int N>
__global__ void __launch_bounds__(kPackThreads) pack_wide_kernel(const T* rows, long long row_stride, long long n, int d,
                                                                 int group, unsigned char* codes, __nv_bfloat16* scales) {
  next_launch_may_start();
  wait_for_launch_before();
  const int lane = lane_id();
  const long long row = (long long)blockIdx.x * (kPackThreads / 32) + (threadIdx.x >> 5);
  if (row >= n) return;
  const T* src = rows + row * row_stride;
  const int blocks = (d + kBlock - 1) / kBlock, words = 4 * blocks, group_words = group / 8, groups = (d + group - 1) / group;
  for (int g = 0; g < groups; ++g) {
    const int first = g * group_words, until = min(first + group_words, words);
    float most = 0.0f;
    T v[8];
    for (int w = first + lane; w < until; w += 32) {
      load_eight<T, N>(src, 8 * w, d, v);
      most = largest(v, most);
    }
    for (int off = 1; off < 32; off <<= 1) most = max_or_nan(most, __shfl_xor_sync(FULL, most, off));
    const __nv_bfloat16 scale = scale_of(most);
    for (int w = first + lane; w < until; w += 32) {
      load_eight<T, N>(src, 8 * w, d, v);
      const float step = __bfloat162float(scale);
      const unsigned word = ordinary(step) ? codes_of(v, step) : codes_of_any(v, step);
      *reinterpret_cast<unsigned*>(codes + row * (16ll * blocks) + word_offset(w, blocks)) = word;
    }
    if (lane == 0) scales[row * groups + g] = scale;
  }
}

// `lanes` threads share `each` rows, V neighbouring values of each (V divides 8): where they are in a row is worked out once.  kRows
// rows are on their way at a time.
// Bound: HBM bytes (50 000 rows of 2048 to fp32 in 77 us, 6.0 TB/s).  Eight rows on their way: 1 000 000 of 51 floats, caches cold, 74 us,
// with 4 102, with 16 88; 50 000 of 2048 80, 82 and 78.
template <class T, int V, int kRows>
__global__ void __launch_bounds__(kPackThreads) unpack_kernel(const unsigned char* codes, const __nv_bfloat16* scales,
                                                              long long n, int d, int group, int group_shift, T* out,
                                                              int lanes, int each) {
  next_launch_may_start();
  wait_for_launch_before();
  const int lane = threadIdx.x & (lanes - 1);
  const long long first = ((long long)blockIdx.x * (kPackThreads / lanes) + threadIdx.x / lanes) * each;
  const int rows = (int)min((long long)each, n - first);
  const int blocks = (d + kBlock - 1) / kBlock, groups = (d + group - 1) / group, row_bytes = 16 * blocks;
  for (int dim = lane * V; dim < d; dim += lanes * V) {
    const unsigned char* word_at = codes + first * row_bytes + word_offset(dim >> 3, blocks);
    const __nv_bfloat16* scale_at = scales + first * groups + (group_shift >= 0 ? dim >> group_shift : dim / group);
    T* to = out + first * d + dim;
    auto pass = [&](auto count) {
      constexpr int kCount = decltype(count)::value;
      unsigned word[kCount];
      __nv_bfloat16 scale[kCount];
#pragma unroll
      for (int r = 0; r < kCount; ++r) {
        word[r] = *reinterpret_cast<const unsigned*>(word_at);
        scale[r] = *scale_at;
        word_at += row_bytes;
        scale_at += groups;
      }
#pragma unroll
      for (int r = 0; r < kCount; ++r) {
        T v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int k = (V == 8 ? 0 : dim & 7) + i;
          // 2^23 + code, and 2^23 + 8 taken away: exact
          const float code = __uint_as_float(((word[r] >> (4 * ((k >> 1) + 4 * (k & 1)))) & 15) | 0x4b000000u) - 8388616.0f;
          v[i] = from_f32<T>(code * __bfloat162float(scale[r]));
        }
        store_many<T, V>(to, v);
        to += d;
      }
    };
    int r = 0;
    for (; r + kRows <= rows; r += kRows) pass(std::integral_constant<int, kRows>());
    for (; r < rows; ++r) pass(std::integral_constant<int, 1>());
  }
}

template <class T, int N>
cudaError_t pack_n(const T* rows, long long row_stride, long long n, int d, long long group, void* codes, void* scales,
                   cudaStream_t stream) {
  const int words = 4 * ((d + kBlock - 1) / kBlock);
  const int lanes = next_pow2(words, 32);
  unsigned char* c = static_cast<unsigned char*>(codes);
  __nv_bfloat16* s = static_cast<__nv_bfloat16*>(scales);
  if (group / 8 > lanes && words > lanes) {
    const long long blocks = (n + kPackThreads / 32 - 1) / (kPackThreads / 32);
    if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
    return launch_early(pack_wide_kernel<T, N>, dim3((unsigned)blocks), kPackThreads, 0, stream, rows, row_stride, n, d,
                        (int)group, c, s);
  }
  // a group that is longer than the row is as good as one of all its words
  const int group_words = group / 8 > lanes ? lanes : (int)(group / 8);
  int shift = 0;
  while ((1 << shift) < group_words) ++shift;
  const int teams = kPackThreads / lanes, groups = (int)((d + group - 1) / group);
  // four rows at a time, unless that leaves SMs without work (1 183 514 rows of 50 floats 60 us, one at a
  // time 73; 20 000 of 64 are 4.4 and 4.0)
  const bool longer = words > lanes, many = longer || n > (long long)4 * kSMs * teams;
  const long long per = longer || !many ? teams : 4 * teams, blocks = (n + per - 1) / per;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  if (longer)  // (blocks of a warp per row)
    return launch_early(pack_long_kernel<T, N>, dim3((unsigned)blocks), kPackThreads, 0, stream, rows, row_stride, n, d, shift,
                        groups, c, s);
  auto* kernel = many ? pack_kernel<T, N, 4> : pack_kernel<T, N, 1>;
  return launch_early(kernel, dim3((unsigned)blocks), kPackThreads, 0, stream, rows, row_stride, n, d, shift, groups, c, s, lanes);
}

template <class T>
cudaError_t pack_t(const T* rows, long long row_stride, long long n, long long d, long long group, void* codes,
                   void* scales, cudaStream_t stream) {
  const int w = word_bytes(reinterpret_cast<uintptr_t>(rows) | (unsigned long long)(row_stride * sizeof(T)) |
                           (unsigned long long)(d * sizeof(T)));
  if (w == 16) return pack_n<T, 16 / sizeof(T)>(rows, row_stride, n, (int)d, group, codes, scales, stream);
  if (w == 8) return pack_n<T, 8 / sizeof(T)>(rows, row_stride, n, (int)d, group, codes, scales, stream);
  if (w == 4) return pack_n<T, 4 / sizeof(T)>(rows, row_stride, n, (int)d, group, codes, scales, stream);
  return pack_n<T, 1>(rows, row_stride, n, (int)d, group, codes, scales, stream);
}

template <class T, int V>
cudaError_t unpack_v(const unsigned char* codes, const __nv_bfloat16* scales, long long n, int d, int group, T* out,
                     cudaStream_t stream) {
  const int lanes = next_pow2((d + V - 1) / V, kPackThreads);
  // 16 rows, fewer while there are not four CTAs per SM (1 183 514 rows of 50 dimensions 59 us, one at a time 246)
  int each = 16;
  while (each > 1 && n / ((long long)(kPackThreads / lanes) * each) < 4 * kSMs) each /= 2;
  const long long per = (long long)(kPackThreads / lanes) * each, blocks = (n + per - 1) / per;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  int shift = 0;
  while ((1 << shift) < group) ++shift;
  auto* kernel = each >= 8   ? unpack_kernel<T, V, 8>
                 : each == 4 ? unpack_kernel<T, V, 4>
                 : each == 2 ? unpack_kernel<T, V, 2>
                             : unpack_kernel<T, V, 1>;
  return launch_early(kernel, dim3((unsigned)blocks), kPackThreads, 0, stream, codes, scales, n, d, group,
                      (1 << shift) == group ? shift : -1, out, lanes, each);
}

template <class T>
cudaError_t unpack_t(const void* codes, const void* scales, long long n, long long d, long long group, void* out,
                     cudaStream_t stream) {
  const unsigned char* c = static_cast<const unsigned char*>(codes);
  const __nv_bfloat16* s = static_cast<const __nv_bfloat16*>(scales);
  T* to = static_cast<T*>(out);
  const int w = word_bytes(reinterpret_cast<uintptr_t>(out) | (unsigned long long)(d * sizeof(T)));
  if (w == 16) return unpack_v<T, 16 / sizeof(T)>(c, s, n, (int)d, (int)group, to, stream);
  if (w == 8) return unpack_v<T, 8 / sizeof(T)>(c, s, n, (int)d, (int)group, to, stream);
  if (w == 4) return unpack_v<T, 4 / sizeof(T)>(c, s, n, (int)d, (int)group, to, stream);
  return unpack_v<T, 1>(c, s, n, (int)d, (int)group, to, stream);
}

// ---- products -------------------------------------------------------------------------------------------------------

// y[q, r] = sum over groups of scale[r, g] * (sum over the group's dimensions of (code - 8) * x[q, i])
//
// The rows are the first operand of the matrix instruction (16 rows x 16 dimensions), the queries the second (8 columns): a
// code becomes a half or bfloat16 value exactly, and so do products and the sums of a group in fp32; the scale is applied to
// a group's sum in fp32.  An fp32 query is three columns of bfloat16, 8 bits of it each, whose sums are added at the end.
//
// Bound: HBM bytes of the codes while the columns are few, then instructions.  A warp has 32 or 16 rows and a share of their
// dimensions; the codes of its next 128 dimensions, of its next rows behind the last ones, are on their way in registers while
// it multiplies these.  A CTA's warps are `split` shares x warps/split sets of rows; all of them read the queries in shared memory.
constexpr int kMostScoreWarps = 16;  // of a CTA that has an SM for itself
// A warp takes 32 rows where that leaves 16 warps the registers for its sums, of up to two tiles of columns, and 16 rows else.
// (131 072 x 4096, 32 queries: 154 us with 16 rows and 16 warps, 156 with 16 and 20, 166 with 32 and 12; 16 queries and 8192
// dimensions: 60 with 32 rows, 67 with 16.)
template <int kTiles>
struct ScoreShape {
  static constexpr int kRowTiles = kTiles >= 3 ? 1 : 2;  // operands of 16 rows per warp
  static constexpr int kWarpRows = 16 * kRowTiles;
  static constexpr int kRowsPerLane = 2 * kRowTiles;     // of the first operand: rows g, g + 8, ..
  static constexpr int kSumPitch = kWarpRows + 1;
};

__device__ __forceinline__ void copy_async(unsigned to, const void* from) {  // 16 bytes
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

struct ScoreLayout {
  int queries;       // of a tile of columns: at most 8 * kTiles / parts
  int pitch;         // values per column of a buffer of queries in shared memory
  int chunk_fours;   // fours of blocks whose queries are in a buffer: all of them, or there are two buffers in turn
  int chunks;
  int split;         // warps that share the same rows, of every chunk
  int column_tiles;
  int wide_queries;  // 16-byte loads of queries
  int wide_scales;   // loads of all scales of four blocks at once
};

// The queries' values of the fours [first, first + count) to shared memory, zeros behind the last dimension.  Values that need
// no change are copied asynchronously (`later`: the caller waits).
template <class Columns>
__device__ __forceinline__ void stage_queries(const Scores4Params& p, const ScoreLayout& l, long long q0, int nq, int first,
                                              int count, bool later, unsigned short* xs) {
  using In = typename Columns::In;
  const int eights = count * (kFour / 8), warps = blockDim.x >> 5;
  const In* queries = static_cast<const In*>(p.queries) + q0 * p.query_stride + (long long)first * kFour;
  const long long left = p.d - (long long)first * kFour;
  auto eight = [&](const In* src, unsigned short* to, int i) {
    const bool whole = l.wide_queries && 8 * i + 8 <= left;
    if constexpr (Columns::kParts == 1) {
      if (later && whole) {
        copy_async((unsigned)__cvta_generic_to_shared(to + 8 * i), src + 8 * i);
        return;
      }
    }
    In v[8];
    if (whole) {
      load_many<In, 8>(src + 8 * i, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 8 * i + j < left ? src[8 * i + j] : from_f32<In>(0.0f);
    }
#pragma unroll
    for (int c = 0; c < Columns::kParts; ++c) {
      unsigned w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = (unsigned)Columns::part(v[2 * j], c) | ((unsigned)Columns::part(v[2 * j + 1], c) << 16);
      *reinterpret_cast<uint4*>(to + c * nq * l.pitch + 8 * i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  };
  if (nq * 2 > warps) {  // a warp per query
    for (int q = threadIdx.x >> 5; q < nq; q += warps) {
      const In* src = queries + q * p.query_stride;
      unsigned short* to = xs + q * l.pitch;
      for (int i = lane_id(); i < eights; i += 32) eight(src, to, i);
    }
  } else {  // all warps for each query
    for (int q = 0; q < nq; ++q)
      for (int i = threadIdx.x; i < eights; i += blockDim.x) eight(queries + q * p.query_stride, xs + q * l.pitch, i);
  }
}

// kGroup: blocks of 32 dimensions per scale, 4 for four and more.  The parts of an fp32 query are the same column of three
// operands, so that a lane holds all its sums.
template <class Columns, int kTiles, int kGroup>
__global__ void __launch_bounds__(32 * kMostScoreWarps, 1) scores_kernel(const __grid_constant__ Scores4Params p,
                                                                      const __grid_constant__ ScoreLayout l) {
  using Pairs = typename Columns::Pairs;
  constexpr int kOutTiles = kTiles / Columns::kParts;
  constexpr int kRowTiles = ScoreShape<kTiles>::kRowTiles, kWarpRows = ScoreShape<kTiles>::kWarpRows;
  constexpr int kRowsPerLane = ScoreShape<kTiles>::kRowsPerLane, kSumPitch = ScoreShape<kTiles>::kSumPitch;
  extern __shared__ __align__(16) unsigned char smem[];
  next_launch_may_start();
  wait_for_launch_before();
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = lane_id(), g = lane >> 2, t = lane & 3;
  const int part = warp % l.split, set = warp / l.split, sets = warps / l.split;
  // the tiles of columns of the same rows run side by side: the second one finds the codes in the L2 cache
  const long long q0 = (long long)(blockIdx.x % l.column_tiles) * l.queries;
  const int nq = (int)min((long long)l.queries, p.nq - q0);
  const int first_unit = blockIdx.x / l.column_tiles, step = gridDim.x / l.column_tiles;
  // shared memory: the sums on their way out [warp][8 columns][row], the queries
  float* sums = reinterpret_cast<float*>(smem);
  unsigned short* xs = reinterpret_cast<unsigned short*>(sums + warps * 8 * kSumPitch);
  const int buffer = l.queries * Columns::kParts * l.pitch;  // of the second buffer of queries
  const int blocks = (int)((p.d + kBlock - 1) / kBlock), fours = (blocks + 3) / 4;
  const int groups = (int)packed_groups_device(p.d, p.group), group_fours = (int)(p.group / kFour);
  const int row_bytes = 16 * blocks;
  const unsigned rows = (unsigned)p.n;
  const int units = (int)((p.n + kWarpRows * sets - 1) / (kWarpRows * sets));
  // a warp's last rows are the table's last ones: some of them are another warp's as well, which writes them
  const unsigned last_start = max(rows, (unsigned)kWarpRows) - kWarpRows;
  auto first_row = [&](int unit) { return min((unsigned)(unit * sets + set) * kWarpRows, last_start); };
  int row_at[kRowsPerLane];
#pragma unroll
  for (int i = 0; i < kRowsPerLane; ++i) row_at[i] = (int)min((unsigned)(g + 8 * i), rows - 1) * row_bytes + 16 * t;
  // The lanes of a row load the scales of a row each, t those of row g + 8 * t; of two rows and four scales, two each.
  constexpr bool kHalves = kGroup == 1 && kRowsPerLane == 2;
  const int half = kHalves ? 2 * (t >> 1) : 0;
  const int scale_at = (int)min((unsigned)(g + 8 * (t % kRowsPerLane)), rows - 1) * groups + half;
  const Pairs pairs;

  // The way through the rows: the fours of this warp's share of every chunk, unit after unit, one ahead of the sums.
  const int share = (l.chunk_fours + l.split - 1) / l.split, first_four = part * share;
  int ahead_unit = first_four < min(l.chunk_fours, fours) ? first_unit : units;
  int ahead_four = first_four, ahead_left = min(share, fours - first_four);  // until the share of this chunk ends
  const unsigned char* src = nullptr;
  const unsigned short* scale_src = nullptr;
  uint4 next_words[kRowsPerLane];
  FourScales<kHalves ? 2 : kGroup> next_scale;
  auto start_unit = [&] {
    src = static_cast<const unsigned char*>(p.codes) + (long long)first_row(ahead_unit) * row_bytes + 64 * ahead_four;
    scale_src = static_cast<const unsigned short*>(p.scales) + (long long)first_row(ahead_unit) * groups + scale_at;
  };
  if (ahead_unit < units) start_unit();
  auto load = [&] {
    if (ahead_unit < units) {
      if (4 * ahead_four + 4 <= blocks) {
#pragma unroll
        for (int i = 0; i < kRowsPerLane; ++i) next_words[i] = __ldcs(reinterpret_cast<const uint4*>(src + row_at[i]));
      } else {
        const int m = blocks - 4 * ahead_four;
        const unsigned char* from = src + 4 * t * m - 16 * t;
#pragma unroll
        for (int i = 0; i < kRowsPerLane; ++i) {
          // (whatever the blocks behind the last one hold: their queries are zeros)
          const unsigned* w = reinterpret_cast<const unsigned*>(from + row_at[i]);
          next_words[i] = make_uint4(w[0], m > 1 ? w[1] : 0, m > 2 ? w[2] : 0, 0);
        }
      }
      const int at = kGroup < 4 ? ahead_four * (4 / kGroup) : group_fours == 1 ? ahead_four : ahead_four / group_fours;
      next_scale.load(scale_src + at, groups - at - half, l.wide_scales);
      ++ahead_four;
      src += 64;
      if (--ahead_left == 0) {
        ahead_four += l.chunk_fours - share;
        src += 64 * (l.chunk_fours - share);
        if (ahead_four >= fours) {
          ahead_four = first_four;
          ahead_unit += step;
          if (ahead_unit < units) start_unit();
        }
        ahead_left = min(share, fours - ahead_four);
      }
    }
  };
  load();
  stage_queries<Columns>(p, l, q0, nq, 0, min(l.chunk_fours, fours), false, xs);

  // lanes of columns that there are not read the last one's and throw the result away
  int column[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i)
    column[i] = (Columns::kParts == 1 ? min(8 * i + g, nq - 1) : i * nq + min(g, nq - 1)) * l.pitch + 8 * t;
  int current = 0;  // buffer of the queries
  __syncthreads();

  for (int unit = first_unit; unit < units; unit += step) {
    float bias[kRowsPerLane];  // of a warp that has its rows for itself
#pragma unroll
    for (int i = 0; i < kRowsPerLane; ++i) {
      const unsigned row = first_row(unit) + g + 8 * i;
      bias[i] = p.bias && l.split == 1 && row < rows ? p.bias[row] : 0.0f;
    }
    float total[kRowTiles][kTiles][4];
#pragma unroll
    for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) total[r][i][j] = 0.0f;
    for (int chunk = 0; chunk < l.chunks; ++chunk) {
      const int base = chunk * l.chunk_fours;
      const int from = base + first_four, to = min(min(fours, base + l.chunk_fours), from + share);
      if (l.chunks > 1 && (chunk + 1 < l.chunks || unit + step < units)) {
        const int next = chunk + 1 < l.chunks ? base + l.chunk_fours : 0;
        stage_queries<Columns>(p, l, q0, nq, next, min(l.chunk_fours, fours - next), true, xs + (current ^ 1) * buffer);
        copies_end();
      }
      const unsigned short* values = xs + current * buffer + first_four * kFour;
#pragma unroll 1
      for (int four = from; four < to; ++four, values += kFour) {
        uint4 w[kRowsPerLane];
        FourScales<kGroup> use[kRowsPerLane];
#pragma unroll
        for (int i = 0; i < kRowsPerLane; ++i) {
          w[i] = next_words[i];
          if constexpr (kHalves) {
            use[i].low = next_scale.of_lane((lane & ~3) + i).low;
            use[i].high = next_scale.of_lane((lane & ~3) + i + 2).low;
          } else {
            use[i] = next_scale.of_lane((lane & ~3) + i);
          }
        }
        load();
        float sum[kRowTiles][kTiles][4];
        auto block = [&](int j) {
          uint4 b[kTiles];
#pragma unroll
          for (int i = 0; i < kTiles; ++i) b[i] = *reinterpret_cast<const uint4*>(values + column[i] + j * kBlock);
#pragma unroll
          for (int r = 0; r < kRowTiles; ++r) {
            const uint4& low = w[2 * r];
            const uint4& high = w[2 * r + 1];
            const unsigned wa = j == 0 ? low.x : j == 1 ? low.y : j == 2 ? low.z : low.w;
            const unsigned wb = j == 0 ? high.x : j == 1 ? high.y : j == 2 ? high.z : high.w;
            const unsigned a0[4] = {pairs.template values<0>(wa), pairs.template values<0>(wb),
                                    pairs.template values<1>(wa), pairs.template values<1>(wb)};
            const unsigned a1[4] = {pairs.template values<2>(wa), pairs.template values<2>(wb),
                                    pairs.template values<3>(wa), pairs.template values<3>(wb)};
#pragma unroll
            for (int i = 0; i < kTiles; ++i) Pairs::mma(sum[r][i], a0, b[i].x, b[i].y, j % kGroup == 0);
#pragma unroll
            for (int i = 0; i < kTiles; ++i) Pairs::mma(sum[r][i], a1, b[i].z, b[i].w, false);
          }
        };
        auto add = [&](int j) {
#pragma unroll
          for (int r = 0; r < kRowTiles; ++r) {
            const float fa = use[2 * r].get(j / kGroup), fb = use[2 * r + 1].get(j / kGroup);
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
              total[r][i][0] += fa * sum[r][i][0];
              total[r][i][1] += fa * sum[r][i][1];
              total[r][i][2] += fb * sum[r][i][2];
              total[r][i][3] += fb * sum[r][i][3];
            }
          }
        };
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          block(j);
          if ((j + 1) % kGroup == 0) add(j);
        }
      }
      if (l.chunks > 1) {
        copies_wait();
        __syncthreads();
        current ^= 1;
      }
    }
    auto value = [&](int i, int r, int c) {
      float y = total[r / 2][i * Columns::kParts][2 * (r % 2) + c];
      if constexpr (Columns::kParts == 3)
        y += total[r / 2][i * Columns::kParts + 1][2 * (r % 2) + c] + total[r / 2][i * Columns::kParts + 2][2 * (r % 2) + c];
      return y;
    };
    if (l.split == 1) {
      // eight rows of four queries at a time
      const unsigned row0 = first_row(unit) + g;
#pragma unroll
      for (int i = 0; i < kOutTiles; ++i) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int q = 8 * i + 2 * t + c;
          if (q < nq) {
            float* out = p.out + (q0 + q) * p.n + row0;
#pragma unroll
            for (int r = 0; r < kRowsPerLane; ++r)
              if (row0 + 8 * r < rows) out[8 * r] = value(i, r, c) + bias[r];
          }
        }
      }
    } else {
      // through shared memory, eight queries at a time: rows next to each other, the shares added up
      float* mine = sums + warp * 8 * kSumPitch;
#pragma unroll
      for (int i = 0; i < kOutTiles; ++i) {
        const int some = min(8, nq - 8 * i);
        if (some <= 0) break;
#pragma unroll
        for (int r = 0; r < kRowsPerLane; ++r)
#pragma unroll
          for (int c = 0; c < 2; ++c) mine[(2 * t + c) * kSumPitch + g + 8 * r] = value(i, r, c);
        float* out = p.out + (q0 + 8 * i) * p.n;
        __syncthreads();
        // a warp takes a set's rows of one column at a time
        for (int k = warp; k < some * sets; k += warps) {
          const int q = k / sets, s = k % sets;
          const unsigned nominal = (unsigned)(unit * sets + s) * kWarpRows;
          const unsigned row = min(nominal, last_start) + lane;
          if (lane < kWarpRows && row < rows && row >= nominal) {
            const float* of_set = sums + (s * l.split * 8 + q) * kSumPitch + lane;
            float y = of_set[0];
            for (int other = 1; other < l.split; ++other) y += of_set[other * 8 * kSumPitch];
            out[q * p.n + row] = y + (p.bias ? p.bias[row] : 0.0f);
          }
        }
        __syncthreads();
      }
    }
  }
  copies_wait();
}

template <class Columns, int kTiles, int kGroup>
cudaError_t scores_t(const Scores4Params& p, int queries, cudaStream_t stream) {
  constexpr int kWarpRows = ScoreShape<kTiles>::kWarpRows, kSumPitch = ScoreShape<kTiles>::kSumPitch;
  constexpr int kMostSpace = 224 * 1024, kHalfSpace = 112 * 1024;  // shared memory of one CTA per SM, of each of two
  ScoreLayout l;
  l.queries = (int)(p.nq < queries ? p.nq : queries);
  const int columns = l.queries * Columns::kParts;
  const int fours = (int)((p.d + kFour - 1) / kFour);
  l.column_tiles = (int)((p.nq + l.queries - 1) / l.queries);
  auto space = [&](int warps, int in_chunk) {
    // eight lanes read 16 bytes of two columns and four parts: half a row of banks from column to column
    return (size_t)columns * (in_chunk * kFour + 32) * 2 * (in_chunk < fours ? 2 : 1) +
           (size_t)warps * 8 * kSumPitch * 4;
  };
  // two CTAs of eight warps per SM, or one of as many as the queries leave room for; queries that do not fit pass through
  // shared memory in chunks, for all warps of a CTA together
  const long long sets = (p.n + kWarpRows - 1) / kWarpRows;
  int warps = 8, per_sm = 2;
  l.chunk_fours = fours;
  if (kTiles >= 3 || space(8, fours) > kHalfSpace) {
    per_sm = 1;
    warps = kMostScoreWarps;
    while (warps > 8 && space(warps, fours) > kMostSpace) warps -= 4;
    if (space(warps, fours) > kMostSpace) {
      warps = kMostScoreWarps;
      l.chunk_fours = 4;
    }
  }
  // How many warps share the same rows, and how many an SM's only CTA has: what takes the CTA with the most units the least time, in
  // steps of four blocks of all its warps.  The end of a unit takes about two of them, four where sums of several warps are
  // added up; chunks of queries are as many bytes as the codes of `columns` rows, for fewer rows the more warps share them.
  const long long room = ((long long)kSMs * per_sm + l.column_tiles - 1) / l.column_tiles;
  const bool chunked = l.chunk_fours < fours;
  const int most_warps = warps;
  long long least = 0;
  for (int w = most_warps; w >= (per_sm == 1 ? 8 : 6); --w) {
    for (int split = 1; split <= 8 && split <= fours; split *= 2) {
      if (w % split != 0 || (chunked && (split > 4 || space(w, 4 * split) > kMostSpace))) continue;
      const long long units = (sets + w / split - 1) / (w / split), steps = (fours + split - 1) / split;
      const long long time = (units + room - 1) / room * w *
                             (steps + (chunked ? steps * columns * split / (32 * w) : 0) + (split == 1 ? 2 : 4));
      // (fewer warps hide less: only for a gain of a twentieth)
      if (least == 0 || (w == warps ? time < least : 20 * time < 19 * least)) {
        least = time;
        l.split = split;
        warps = w;
      }
    }
  }
  if (chunked) l.chunk_fours = 4 * l.split;
  l.chunks = (fours + l.chunk_fours - 1) / l.chunk_fours;
  l.pitch = l.chunk_fours * kFour + 32;
  const size_t smem = space(warps, l.chunk_fours);
  const long long units = (sets + warps / l.split - 1) / (warps / l.split);
  const long long step = room < units ? room : units;
  if (step * l.column_tiles > 0x7fffffffll) return cudaErrorInvalidValue;
  l.wide_queries = word_bytes(reinterpret_cast<uintptr_t>(p.queries) |
                              (unsigned long long)(p.query_stride * sizeof(typename Columns::In))) == 16;
  const int per_four = kGroup == 1 ? 4 : kGroup == 2 ? 2 : 1;
  l.wide_scales = packed_groups(p.d, p.group) % per_four == 0 && reinterpret_cast<uintptr_t>(p.scales) % (2 * per_four) == 0;
  cudaError_t e = allow_smem<scores_kernel<Columns, kTiles, kGroup>>();
  if (e != cudaSuccess) return e;
  return launch_early(scores_kernel<Columns, kTiles, kGroup>, dim3((unsigned)(step * l.column_tiles)), 32 * warps, smem, stream,
                      p, l);
}

template <class Columns, int kTiles>
cudaError_t scores_group(const Scores4Params& p, int queries, cudaStream_t stream) {
  if (p.group == kBlock) return scores_t<Columns, kTiles, 1>(p, queries, stream);
  if (p.group == 2 * kBlock) return scores_t<Columns, kTiles, 2>(p, queries, stream);
  return scores_t<Columns, kTiles, 4>(p, queries, stream);
}

template <class Columns>
cudaError_t scores_columns(const Scores4Params& p, cudaStream_t stream) {
  // as many queries at a time as the operands have columns, in tiles of equal size
  long long queries = Columns::kParts == 1 ? 32 : 8, tiles = (p.nq + queries - 1) / queries;
  if constexpr (Columns::kParts == 3) {
    // fp32 queries are taken apart on their way into shared memory, for each chunk again where they do not fit.  With few rows,
    // smaller tiles that do fit are better: their rows find idle warps.  (8 queries of 5000 dimensions, 3000 rows: two tiles 18
    // us, chunks 28; 9000 rows: 50 and 39.)
    constexpr long long kSpace = 208 * 1024;
    const long long fit = kSpace / (Columns::kParts * 2 * ((p.d + kFour - 1) / kFour * kFour + 32));
    const long long smaller = fit > 0 ? (p.nq + fit - 1) / fit : 0, sets = (p.n + 15) / 16;
    if (fit >= 4 && fit < 8 && smaller * sets <= 4 * kSMs) tiles = smaller;
  }
  queries = (p.nq + tiles - 1) / tiles;
  if constexpr (Columns::kParts == 3) {
    return scores_group<Columns, 3>(p, (int)queries, stream);
  } else {
    if (queries <= 8) return scores_group<Columns, 1>(p, (int)queries, stream);
    if (queries <= 16) return scores_group<Columns, 2>(p, (int)queries, stream);
    if (queries <= 24) return scores_group<Columns, 3>(p, (int)queries, stream);
    return scores_group<Columns, 4>(p, (int)queries, stream);
  }
}

}  // namespace

cudaError_t launch_pack4(const void* rows, long long row_stride, int type, long long n, long long d, long long group,
                         void* codes, void* scales, cudaStream_t stream) {
  if (n <= 0 || d <= 0) return cudaSuccess;
  if (type == kF32) return pack_t(static_cast<const float*>(rows), row_stride, n, d, group, codes, scales, stream);
  if (type == kF16) return pack_t(static_cast<const __half*>(rows), row_stride, n, d, group, codes, scales, stream);
  return pack_t(static_cast<const __nv_bfloat16*>(rows), row_stride, n, d, group, codes, scales, stream);
}

cudaError_t launch_unpack4(const void* codes, const void* scales, long long n, long long d, long long group, void* out,
                           int type, cudaStream_t stream) {
  if (n <= 0 || d <= 0) return cudaSuccess;
  if (type == kF32) return unpack_t<float>(codes, scales, n, d, group, out, stream);
  if (type == kF16) return unpack_t<__half>(codes, scales, n, d, group, out, stream);
  return unpack_t<__nv_bfloat16>(codes, scales, n, d, group, out, stream);
}

cudaError_t launch_scores4(const Scores4Params& p, cudaStream_t stream) {
  if (p.n <= 0 || p.nq <= 0) return cudaSuccess;
  if (p.d <= kFour) return launch_scores4_narrow(p, stream);  // (both sides measured there)
  if (p.type == kF32) return scores_columns<ColumnsF32>(p, stream);
  if (p.type == kF16) return scores_columns<ColumnsF16>(p, stream);
  return scores_columns<ColumnsBF16>(p, stream);
}

}  // namespace hnsw
