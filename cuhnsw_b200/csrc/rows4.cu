// Rows of a table in 4 bits: packing, unpacking, and products of queries with all rows.
//
// A value is (code - 8) * scale: a code of 0..15 per value and a bfloat16 scale per `group` consecutive dimensions of a row.
// A row's codes are 32-bit words of eight values (16 bytes per block of 32 dimensions, the last one filled up with code 8).
// Blocks lie in fours (the last of a row as many as are left, m): word t*m + j of a four holds dimensions 8t..8t+7 of its
// block j, the even ones in nibbles 0..3, the odd ones in nibbles 4..7.  So a lane's 16 bytes of a row are its part of four
// steps of the matrix instruction over 32 dimensions each, a group of 32 or 64 dimensions ends between two steps, and
// w & 0x000f000f is a pair of consecutive values in two halves of a register.
#include "common.cuh"
#include "table_common.cuh"

namespace hnsw {

namespace {

constexpr int kBlock = 32;             // dimensions of a block
constexpr int kFour = 4 * kBlock;      // of four blocks

__device__ __forceinline__ long long packed_groups_device(long long d, long long group) { return (d + group - 1) / group; }

// Byte offset in a row of the word that holds dimensions 8 * index .. 8 * index + 7
__device__ __forceinline__ long long word_offset(long long index, long long blocks) {
  const long long four = index / 16, block = index / 4, t = index % 4;
  const int m = (int)min(4ll, blocks - 4 * four);
  return 64 * four + 4 * (t * m + (block - 4 * four));
}

// ---- packing --------------------------------------------------------------------------------------------------------

constexpr int kPackThreads = 256;

template <class T, int N>
__device__ __forceinline__ void load_eight(const T* row, long long dim, long long d, float (&v)[8]) {
  if (dim + 8 <= d) {
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      T w[N];
      load_many<T, N>(row + dim + i, w);
#pragma unroll
      for (int j = 0; j < N; ++j) v[i + j] = to_f32(w[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = dim + i < d ? to_f32(row[dim + i]) : 0.0f;
  }
}

// `lanes` lanes (a power of two, at most a warp) share a row, eight dimensions each at a time.  Bound: HBM bytes.
template <class T, int N>
__global__ void __launch_bounds__(kPackThreads) pack_kernel(const T* rows, long long row_stride, long long n, long long d,
                                                            long long group, unsigned char* codes,
                                                            __nv_bfloat16* scales, int lanes) {
  const int lane = threadIdx.x % lanes;
  const long long row = (long long)blockIdx.x * (kPackThreads / lanes) + threadIdx.x / lanes;
  if ((threadIdx.x & ~31) / lanes + (long long)blockIdx.x * (kPackThreads / lanes) >= n) return;  // the whole warp
  const bool live = row < n;
  const T* src = rows + (live ? row : 0) * row_stride;
  const long long blocks = (d + kBlock - 1) / kBlock, words = 4 * blocks, groups = packed_groups_device(d, group);
  unsigned char* dst = codes + row * 16 * blocks;
  const long long group_words = group / 8;
  const int span = (int)min((long long)lanes, group_words);  // lanes that share a group at a time
  for (long long first = 0; first < words; first += group_words > lanes ? group_words : lanes) {
    // the largest magnitude of each group
    const long long until = group_words > lanes ? min(first + group_words, words) : min(first + lanes, words);
    float most = 0.0f, v[8];
    for (long long w = first + lane; w < until; w += lanes) {
      load_eight<T, N>(src, 8 * w, d, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[i]));
    }
    for (int off = 1; off < span; off <<= 1) most = fmaxf(most, __shfl_xor_sync(FULL, most, off));
    const __nv_bfloat16 scale = __float2bfloat16_rn(__fmul_rn(most, 1.0f / 7.0f));
    const float step = __bfloat162float(scale);
    for (long long w = first + lane; w < until; w += lanes) {
      if (until - first > lanes) load_eight<T, N>(src, 8 * w, d, v);
      unsigned word = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float q = step > 0.0f ? fminf(fmaxf(rintf(__fdiv_rn(v[i], step)), -8.0f), 7.0f) : 0.0f;
        const unsigned code = (unsigned)((int)q + 8);
        word |= code << (4 * ((i >> 1) + 4 * (i & 1)));
      }
      if (live) *reinterpret_cast<unsigned*>(dst + word_offset(w, blocks)) = word;
      if (live && w % group_words == 0 && w / group_words < groups) scales[row * groups + w / group_words] = scale;
    }
  }
}

template <class T>
__global__ void __launch_bounds__(kPackThreads) unpack_kernel(const unsigned char* codes, const __nv_bfloat16* scales,
                                                              long long n, long long d, long long group, T* out) {
  const long long blocks = (d + kBlock - 1) / kBlock, words = (d + 7) / 8, groups = packed_groups_device(d, group);
  const long long step = (long long)gridDim.x * kPackThreads;
  for (long long at = (long long)blockIdx.x * kPackThreads + threadIdx.x; at < n * words; at += step) {
    const long long row = at / words, w = at % words;
    const unsigned word = *reinterpret_cast<const unsigned*>(codes + row * 16 * blocks + word_offset(w, blocks));
    const float scale = __bfloat162float(scales[row * groups + 8 * w / group]);
    T* to = out + row * d + 8 * w;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int code = (word >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15;
      if (8 * w + i < d) to[i] = from_f32<T>((float)(code - 8) * scale);
    }
  }
}

template <class T>
cudaError_t pack_t(const T* rows, long long row_stride, long long n, long long d, long long group, void* codes,
                   void* scales, cudaStream_t stream) {
  const int lanes = next_pow2(4 * ((d + kBlock - 1) / kBlock), 32);
  const long long blocks = (n * lanes + kPackThreads - 1) / kPackThreads;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  const int w = word_bytes(reinterpret_cast<uintptr_t>(rows) | (unsigned long long)(row_stride * sizeof(T)));
#define PACK(N) pack_kernel<T, N><<<(unsigned)blocks, kPackThreads, 0, stream>>>( \
    rows, row_stride, n, d, group, static_cast<unsigned char*>(codes), static_cast<__nv_bfloat16*>(scales), lanes)
  if (w == 16)
    PACK(16 / sizeof(T));
  else if (w == 8)
    PACK(8 / sizeof(T));
  else if (w == 4)
    PACK(4 / sizeof(T));
  else
    PACK(1);
#undef PACK
  return cudaGetLastError();
}

// ---- products -------------------------------------------------------------------------------------------------------

// y[q, r] = sum over groups of scale[r, g] * (sum over the group's dimensions of (code - 8) * x[q, i])
//
// The rows are the first operand of the matrix instruction (16 rows x 16 dimensions), the queries the second (8 columns): a
// code becomes a half or bfloat16 value exactly, and so do products and the sums of a group in fp32; the scale is applied to
// a group's sum in fp32.  An fp32 query is three columns of bfloat16, 8 bits of it each, whose sums are added at the end.
//
// Bound: HBM bytes of the codes while the columns are few.  A warp has 32 rows and a share of their dimensions.  It copies its
// codes asynchronously into a ring of its own in shared memory, two steps of 128 dimensions ahead and across the end of its rows, so
// that nothing waits for a barrier to keep the copies going; every lane reads back what it copied itself.  A CTA's warps are
// `split` shares x warps/split sets of 32 rows; all of them read the queries in shared memory.
constexpr int kRowTiles = 2;                  // operands of 16 rows per warp
constexpr int kWarpRows = 16 * kRowTiles;
constexpr int kRowsPerLane = 2 * kRowTiles;   // of the first operand: rows g, g + 8, g + 16, ..
constexpr int kSumPitch = kWarpRows + 1;
constexpr int kStages = 3;                    // of the ring
constexpr int kStageBytes = kWarpRows * 64;
constexpr int kMostScoreThreads = 512;

template <int Bytes>
__device__ __forceinline__ void copy_async(unsigned to, const void* from) {
  if constexpr (Bytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(Bytes) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int Left>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(Left) : "memory"); }

struct PairsF16 {
  // two codes of nibbles `pair` and `pair` + 4 as code - 8
  template <int Pair>
  static __device__ __forceinline__ unsigned values(unsigned w) {
    const unsigned u = Pair >= 2 ? w >> 8 : w;
    if (Pair % 2 == 0) {
      const unsigned v = (u & 0x000f000fu) | 0x64006400u;  // 1024 + code
      const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), __half2half2(__ushort_as_half(0x6408)));
      return *reinterpret_cast<const unsigned*>(&r);
    }
    const unsigned v = (u & 0x00f000f0u) | 0x64006400u;    // 1024 + 16 * code
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&v), __half2half2(__ushort_as_half(0x2c00)),
                              __half2half2(__ushort_as_half(0xd480)));  // / 16 - 72
    return *reinterpret_cast<const unsigned*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
struct PairsBF16 {
  template <int Pair>
  static __device__ __forceinline__ unsigned values(unsigned w) {
    const unsigned v = ((w >> (4 * Pair)) & 0x000f000fu) | 0x43004300u;  // 128 + code
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v),
                                     __bfloat162bfloat162(__ushort_as_bfloat16(0x4308)));
    return *reinterpret_cast<const unsigned*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// How the values of a query type become columns
struct ColumnsF16 {
  using In = __half;
  using Pairs = PairsF16;
  static constexpr int kParts = 1;
  static __device__ __forceinline__ unsigned short part(__half x, int) { return __half_as_ushort(x); }
};
struct ColumnsBF16 {
  using In = __nv_bfloat16;
  using Pairs = PairsBF16;
  static constexpr int kParts = 1;
  static __device__ __forceinline__ unsigned short part(__nv_bfloat16 x, int) { return __bfloat16_as_ushort(x); }
};
struct ColumnsF32 {
  using In = float;
  using Pairs = PairsBF16;
  static constexpr int kParts = 3;
  // x = high + middle + low but for 2^-24 of it: each part is what the ones before leave, rounded to 8 bits
  static __device__ __forceinline__ unsigned short part(float x, int which) {
    const __nv_bfloat16 high = __float2bfloat16_rn(x);
    if (which == 0) return __bfloat16_as_ushort(high);
    // (an infinity or NaN is all in the first part: its remainder would be a NaN)
    const float rest = isfinite(__bfloat162float(high)) ? x - __bfloat162float(high) : 0.0f;
    const __nv_bfloat16 middle = __float2bfloat16_rn(rest);
    return __bfloat16_as_ushort(which == 1 ? middle : __float2bfloat16_rn(rest - __bfloat162float(middle)));
  }
};

struct ScoreLayout {
  int queries;       // of a tile of columns: at most 8 * kTiles / parts
  int pitch;         // values per column in shared memory
  int chunk_fours;   // fours of blocks whose queries are in shared memory at a time
  int split;         // warps that share 32 rows
  int column_tiles;
  int wide_queries;  // 16-byte loads of queries
  int wide_scales;   // loads of all scales of four blocks at once
};

// The queries' values of the dimensions [first, first + count) (a multiple of 8) to shared memory, zeros behind the last one.
template <class Columns>
__device__ __forceinline__ void stage_queries(const Scores4Params& p, const ScoreLayout& l, long long q0, int nq,
                                              long long first, int count, unsigned short* xs) {
  using In = typename Columns::In;
  const In* x = static_cast<const In*>(p.queries);
  const int eights = count / 8;
  for (int q = 0; q < nq; ++q) {
    const In* src = x + (q0 + q) * p.query_stride + first;
    for (int i = threadIdx.x; i < eights; i += blockDim.x) {
      In v[8];
      if (l.wide_queries && first + 8 * i + 8 <= p.d) {
        load_many<In, 8>(src + 8 * i, v);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = first + 8 * i + j < p.d ? src[8 * i + j] : from_f32<In>(0.0f);
      }
#pragma unroll
      for (int c = 0; c < Columns::kParts; ++c) {
        unsigned w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = (unsigned)Columns::part(v[2 * j], c) | ((unsigned)Columns::part(v[2 * j + 1], c) << 16);
        *reinterpret_cast<uint4*>(xs + (c * nq + q) * l.pitch + 8 * i) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

__device__ __forceinline__ float bf16_low(unsigned pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float bf16_high(unsigned pair) { return __uint_as_float(pair & 0xffff0000u); }

// The scales of a row for four blocks: pairs of bfloat16
template <int kGroup>
struct FourScales;
template <>
struct FourScales<1> {
  uint2 raw;
  __device__ __forceinline__ void load(const unsigned short* row, int four, int, int groups, bool wide) {
    if (wide) {
      raw = *reinterpret_cast<const uint2*>(row + 4 * four);
    } else {
      const unsigned short* at = row + 4 * four;
      const int left = groups - 4 * four;
      raw.x = at[0] | (left > 1 ? (unsigned)at[1] << 16 : 0);
      raw.y = (left > 2 ? at[2] : 0) | (left > 3 ? (unsigned)at[3] << 16 : 0);
    }
  }
  __device__ __forceinline__ float get(int j) const {
    return j == 0 ? bf16_low(raw.x) : j == 1 ? bf16_high(raw.x) : j == 2 ? bf16_low(raw.y) : bf16_high(raw.y);
  }
};
template <>
struct FourScales<2> {
  unsigned raw;
  __device__ __forceinline__ void load(const unsigned short* row, int four, int, int groups, bool wide) {
    if (wide)
      raw = *reinterpret_cast<const unsigned*>(row + 2 * four);
    else
      raw = row[2 * four] | (groups - 2 * four > 1 ? (unsigned)row[2 * four + 1] << 16 : 0);
  }
  __device__ __forceinline__ float get(int j) const { return j == 0 ? bf16_low(raw) : bf16_high(raw); }
};
template <>
struct FourScales<4> {
  unsigned raw;
  __device__ __forceinline__ void load(const unsigned short* row, int four, int group_fours, int, bool) {
    raw = row[group_fours == 1 ? four : four / group_fours];
  }
  __device__ __forceinline__ float get(int) const { return bf16_low(raw); }
};

// kGroup: blocks of 32 dimensions per scale, 4 for four and more.  The parts of an fp32 query are the same column of three
// operands, so that a lane holds all its sums.
template <class Columns, int kTiles, int kGroup>
__global__ void __launch_bounds__(kMostScoreThreads, 1) scores_kernel(const __grid_constant__ Scores4Params p,
                                                                      const __grid_constant__ ScoreLayout l) {
  using Pairs = typename Columns::Pairs;
  constexpr int kOutTiles = kTiles / Columns::kParts;
  extern __shared__ __align__(16) unsigned char smem[];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = lane_id(), g = lane >> 2, t = lane & 3;
  const int part = warp % l.split, set = warp / l.split, sets = warps / l.split;
  // the tiles of columns of the same rows run side by side: the second one finds the codes in the L2 cache
  const long long q0 = (long long)(blockIdx.x % l.column_tiles) * l.queries;
  const int nq = (int)min((long long)l.queries, p.nq - q0);
  const int first_unit = blockIdx.x / l.column_tiles, step = gridDim.x / l.column_tiles;
  // shared memory: the rings, the sums on their way out [warp][8 columns][row], the queries
  const unsigned ring = (unsigned)__cvta_generic_to_shared(smem) + warp * (kStages * kStageBytes) + 16 * lane;
  float* sums = reinterpret_cast<float*>(smem + warps * kStages * kStageBytes);
  unsigned short* xs = reinterpret_cast<unsigned short*>(sums + warps * 8 * kSumPitch);
  const int blocks = (int)((p.d + kBlock - 1) / kBlock), fours = (blocks + 3) / 4;
  const int groups = (int)packed_groups_device(p.d, p.group), group_fours = (int)(p.group / kFour);
  const int row_bytes = 16 * blocks;
  const unsigned rows = (unsigned)p.n;
  const unsigned char* codes = static_cast<const unsigned char*>(p.codes);
  const unsigned short* scales = static_cast<const unsigned short*>(p.scales);
  const int units = (int)((p.n + kWarpRows * sets - 1) / (kWarpRows * sets));

  for (int chunk = 0; chunk < fours; chunk += l.chunk_fours) {
    const int in_chunk = min(l.chunk_fours, fours - chunk);
    const int each = (in_chunk + l.split - 1) / l.split;
    const int from = chunk + min(part * each, in_chunk), to = min(chunk + in_chunk, from + each);
    int ahead_unit = first_unit, ahead_four = from;  // what is copied next
    unsigned ahead_slot = 0;
    auto copy = [&] {
      if (ahead_unit < units && from < to) {
        const unsigned row0 = (unsigned)(ahead_unit * sets + set) * kWarpRows + g;
        const int m = min(4, blocks - 4 * ahead_four);
        const int at = 64 * ahead_four + 4 * t * m;
        const unsigned slot = ring + ahead_slot;
#pragma unroll
        for (int i = 0; i < kRowsPerLane; ++i) {
          // rows behind the last one are read as the last one and not written
          const unsigned char* src = codes + (long long)min(row0 + 8 * i, rows - 1) * row_bytes + at;
          if (m == 4) {
            copy_async<16>(slot + 512 * i, src);
          } else if (m == 2) {
            copy_async<8>(slot + 512 * i, src);
          } else {
            copy_async<4>(slot + 512 * i, src);
            if (m == 3) {
              copy_async<4>(slot + 512 * i + 4, src + 4);
              copy_async<4>(slot + 512 * i + 8, src + 8);
            }
          }
        }
        if (++ahead_four == to) {
          ahead_four = from;
          ahead_unit += step;
        }
      }
      ahead_slot = ahead_slot == (kStages - 1) * kStageBytes ? 0 : ahead_slot + kStageBytes;
      copies_end();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) copy();
    if (chunk > 0) __syncthreads();
    stage_queries<Columns>(p, l, q0, nq, (long long)chunk * kFour, in_chunk * kFour, xs);
    __syncthreads();
    // lanes of columns that there are not read the last one's and throw the result away
    const unsigned short* column = xs + 8 * t;

    unsigned slot = 0;
    FourScales<kGroup> scale[kRowsPerLane];
    auto load_scales = [&](int unit, int four) {
      const unsigned row0 = (unsigned)(unit * sets + set) * kWarpRows + g;
#pragma unroll
      for (int i = 0; i < kRowsPerLane; ++i)
        scale[i].load(scales + (long long)min(row0 + 8 * i, rows - 1) * groups, four, group_fours, groups, l.wide_scales);
    };
    if (first_unit < units && from < to) load_scales(first_unit, from);
    for (int unit = first_unit; unit < units; unit += step) {
      float total[kRowTiles][kTiles][4];
#pragma unroll
      for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) total[r][i][j] = 0.0f;
      for (int four = from; four < to; ++four) {
        copy();
        copies_wait<kStages - 1>();
        FourScales<kGroup> now[kRowsPerLane];
#pragma unroll
        for (int i = 0; i < kRowsPerLane; ++i) now[i] = scale[i];
        if (four + 1 < to)
          load_scales(unit, four + 1);
        else if (unit + step < units)
          load_scales(unit + step, from);
        uint4 w[kRowsPerLane];
#pragma unroll
        for (int i = 0; i < kRowsPerLane; ++i)
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                       : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w)
                       : "r"(ring + slot + 512 * i)
                       : "memory");
        slot = slot == (kStages - 1) * kStageBytes ? 0 : slot + kStageBytes;
        const int m = min(4, blocks - 4 * four);
        const unsigned short* values = column + (four - chunk) * kFour;
        float sum[kRowTiles][kTiles][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j % kGroup == 0) {
#pragma unroll
            for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
              for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) sum[r][i][k] = 0.0f;
          }
          if (j < m) {
            uint4 b[kTiles];
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
              const int c = Columns::kParts == 1 ? min(8 * i + g, nq - 1) : i * nq + min(g, nq - 1);
              b[i] = *reinterpret_cast<const uint4*>(values + c * l.pitch + j * kBlock);
            }
#pragma unroll
            for (int r = 0; r < kRowTiles; ++r) {
              const uint4& low = w[2 * r];
              const uint4& high = w[2 * r + 1];
              const unsigned wa = j == 0 ? low.x : j == 1 ? low.y : j == 2 ? low.z : low.w;
              const unsigned wb = j == 0 ? high.x : j == 1 ? high.y : j == 2 ? high.z : high.w;
              const unsigned a0[4] = {Pairs::template values<0>(wa), Pairs::template values<0>(wb),
                                      Pairs::template values<1>(wa), Pairs::template values<1>(wb)};
              const unsigned a1[4] = {Pairs::template values<2>(wa), Pairs::template values<2>(wb),
                                      Pairs::template values<3>(wa), Pairs::template values<3>(wb)};
#pragma unroll
              for (int i = 0; i < kTiles; ++i) {
                Pairs::mma(sum[r][i], a0, b[i].x, b[i].y);
                Pairs::mma(sum[r][i], a1, b[i].z, b[i].w);
              }
            }
          }
          if ((j + 1) % kGroup == 0 && j / kGroup * kGroup < m) {
#pragma unroll
            for (int r = 0; r < kRowTiles; ++r) {
              const float fa = now[2 * r].get(j / kGroup), fb = now[2 * r + 1].get(j / kGroup);
#pragma unroll
              for (int i = 0; i < kTiles; ++i) {
                total[r][i][0] += fa * sum[r][i][0];
                total[r][i][1] += fa * sum[r][i][1];
                total[r][i][2] += fb * sum[r][i][2];
                total[r][i][3] += fb * sum[r][i][3];
              }
            }
          }
        }
      }
      // through shared memory, eight columns at a time: rows next to each other, the shares added up
      float* mine = sums + warp * 8 * kSumPitch;
      const int set_rows = kWarpRows * sets;
#pragma unroll
      for (int i = 0; i < kOutTiles; ++i) {
        const int some = min(8, nq - 8 * i);
        if (some <= 0) break;
#pragma unroll
        for (int r = 0; r < kRowsPerLane; ++r) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float y = total[r / 2][i * Columns::kParts][2 * (r % 2) + c];
            if constexpr (Columns::kParts == 3)
              y += total[r / 2][i * Columns::kParts + 1][2 * (r % 2) + c] +
                   total[r / 2][i * Columns::kParts + 2][2 * (r % 2) + c];
            mine[(2 * t + c) * kSumPitch + g + 8 * r] = y;
          }
        }
        auto write = [&](float y, int q, long long row) {
          float* out = p.out + (q0 + 8 * i + q) * p.n + row;
          if (chunk > 0)
            y += *out;
          else if (p.bias)
            y += p.bias[row];
          *out = y;
        };
        if (l.split == 1) {
          __syncwarp();
          const long long row = (long long)(unit * sets + set) * kWarpRows + lane;
          if (row < p.n)
            for (int q = 0; q < some; ++q) write(mine[q * kSumPitch + lane], q, row);
          __syncwarp();
        } else {
          __syncthreads();
          for (int k = threadIdx.x; k < some * set_rows; k += blockDim.x) {
            const int q = k / set_rows, r = k % set_rows;
            const long long row = (long long)unit * set_rows + r;
            if (row < p.n) {
              const float* of_set = sums + ((r / kWarpRows) * l.split * 8 + q) * kSumPitch + r % kWarpRows;
              float y = of_set[0];
              for (int s = 1; s < l.split; ++s) y += of_set[s * 8 * kSumPitch];
              write(y, q, row);
            }
          }
          __syncthreads();
        }
      }
    }
    copies_wait<0>();
  }
}

template <class Columns, int kTiles, int kGroup>
cudaError_t scores_t(const Scores4Params& p, int queries, cudaStream_t stream) {
  constexpr int kMostSpace = 224 * 1024, kHalfSpace = 112 * 1024;  // shared memory of one CTA per SM, of each of two
  ScoreLayout l;
  l.queries = (int)(p.nq < queries ? p.nq : queries);
  const int columns = l.queries * Columns::kParts;
  const int fours = (int)((p.d + kFour - 1) / kFour);
  auto space = [&](int warps, int in_chunk) {
    // eight lanes read 16 bytes of two columns and four parts: half a row of banks from column to column
    return (size_t)columns * (in_chunk * kFour + 32) * 2 + (size_t)warps * (kStages * kStageBytes + 8 * kSumPitch * 4);
  };
  // two CTAs of eight warps per SM, or one of as many as the queries leave room for
  int warps = 8;
  l.chunk_fours = fours;
  const bool two = space(8, fours) <= kHalfSpace;
  if (!two) {
    warps = 16;
    while (warps > 8 && space(warps, fours) > kMostSpace) warps -= 4;
    while (space(warps, l.chunk_fours) > kMostSpace) l.chunk_fours = (l.chunk_fours + 1) / 2;
  }
  l.pitch = l.chunk_fours * kFour + 32;
  const size_t smem = space(warps, l.chunk_fours);
  l.column_tiles = (int)((p.nq + l.queries - 1) / l.queries);
  // several units for every CTA, and something to do for every warp
  const long long sets = (p.n + kWarpRows - 1) / kWarpRows;
  const long long room = (long long)kSMs * (two ? 2 : 1);
  l.split = 1;
  while (l.split < (warps == 12 ? 4 : 8) && 2 * l.split <= l.chunk_fours &&
         sets * l.split * l.column_tiles < 8 * room * warps)
    l.split *= 2;
  const long long units = (sets + warps / l.split - 1) / (warps / l.split);
  long long step = (room + l.column_tiles - 1) / l.column_tiles;
  if (step > units) step = units;
  if (step * l.column_tiles > 0x7fffffffll) return cudaErrorInvalidValue;
  l.wide_queries = word_bytes(reinterpret_cast<uintptr_t>(p.queries) |
                              (unsigned long long)(p.query_stride * sizeof(typename Columns::In))) == 16;
  const int per_four = kGroup == 1 ? 4 : kGroup == 2 ? 2 : 1;
  l.wide_scales = packed_groups(p.d, p.group) % per_four == 0 && reinterpret_cast<uintptr_t>(p.scales) % (2 * per_four) == 0;
  cudaError_t e = allow_smem<scores_kernel<Columns, kTiles, kGroup>>();
  if (e != cudaSuccess) return e;
  scores_kernel<Columns, kTiles, kGroup><<<(unsigned)(step * l.column_tiles), 32 * warps, smem, stream>>>(p, l);
  return cudaGetLastError();
}

template <class Columns, int kTiles>
cudaError_t scores_group(const Scores4Params& p, int queries, cudaStream_t stream) {
  if (p.group == kBlock) return scores_t<Columns, kTiles, 1>(p, queries, stream);
  if (p.group == 2 * kBlock) return scores_t<Columns, kTiles, 2>(p, queries, stream);
  return scores_t<Columns, kTiles, 4>(p, queries, stream);
}

template <class Columns>
cudaError_t scores_columns(const Scores4Params& p, cudaStream_t stream) {
  // as many queries at a time as fit into the operands' columns and, with all their dimensions, into shared memory; then as many
  // tiles of equal size as that takes
  constexpr long long kSpace = 132 * 1024;
  const long long fit = kSpace / (Columns::kParts * 2 * ((p.d + kFour - 1) / kFour * kFour + 32));
  long long queries = Columns::kParts == 1 ? 32 : 8;
  if (fit < queries) queries = fit < 1 ? 1 : fit;
  const long long tiles = (p.nq + queries - 1) / queries;
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
  const unsigned char* c = static_cast<const unsigned char*>(codes);
  const __nv_bfloat16* s = static_cast<const __nv_bfloat16*>(scales);
  const long long items = n * ((d + 7) / 8);
  const long long wanted = (items + kPackThreads - 1) / kPackThreads, room = kSMs * 32;
  const unsigned blocks = (unsigned)(wanted < room ? wanted : room);
  if (type == kF32)
    unpack_kernel<float><<<blocks, kPackThreads, 0, stream>>>(c, s, n, d, group, static_cast<float*>(out));
  else if (type == kF16)
    unpack_kernel<__half><<<blocks, kPackThreads, 0, stream>>>(c, s, n, d, group, static_cast<__half*>(out));
  else
    unpack_kernel<__nv_bfloat16><<<blocks, kPackThreads, 0, stream>>>(c, s, n, d, group, static_cast<__nv_bfloat16*>(out));
  return cudaGetLastError();
}

cudaError_t launch_scores4(const Scores4Params& p, cudaStream_t stream) {
  if (p.n <= 0 || p.nq <= 0) return cudaSuccess;
  if (p.type == kF32) return scores_columns<ColumnsF32>(p, stream);
  if (p.type == kF16) return scores_columns<ColumnsF16>(p, stream);
  return scores_columns<ColumnsBF16>(p, stream);
}

}  // namespace hnsw
