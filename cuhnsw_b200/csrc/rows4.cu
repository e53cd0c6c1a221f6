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
// Bound: HBM bytes of the codes while the columns are few.  Every warp has 16 rows and a share of their blocks; a CTA's warps
// are `split` shares x 8/split sets of 16 rows.  The queries lie in shared memory.
constexpr int kScoreWarps = 8;
constexpr int kScoreThreads = kScoreWarps * 32;

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
  int columns;      // 8 * kTiles
  int queries;      // of a launch's column tile
  int pitch;        // values per column in shared memory
  int chunk_fours;  // fours of blocks whose queries are in shared memory at a time
  int split;        // warps that share 16 rows
};

template <class Columns, int kTiles>
__global__ void __launch_bounds__(kScoreThreads) scores_kernel(Scores4Params p, ScoreLayout l) {
  using Pairs = typename Columns::Pairs;
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned short* xs = reinterpret_cast<unsigned short*>(smem);
  float* sums = reinterpret_cast<float*>(smem + (size_t)l.columns * l.pitch * 2);  // [warp][column][16 rows + 1]
  const int warp = threadIdx.x >> 5, lane = lane_id(), g = lane >> 2, t = lane & 3;
  const int part = warp % l.split, set = warp / l.split, sets = kScoreWarps / l.split;
  const long long q0 = (long long)blockIdx.y * l.queries;
  const int nq = (int)min((long long)l.queries, p.nq - q0);
  const long long blocks = (p.d + kBlock - 1) / kBlock, row_bytes = 16 * blocks;
  const long long fours = (blocks + 3) / 4, groups = packed_groups_device(p.d, p.group);
  const int group_blocks = (int)min(p.group / kBlock, 1ll << 30);
  const unsigned char* codes = static_cast<const unsigned char*>(p.codes);
  const __nv_bfloat16* scales = static_cast<const __nv_bfloat16*>(p.scales);
  const typename Columns::In* x = static_cast<const typename Columns::In*>(p.queries);
  const long long tiles = (p.n + 16 * sets - 1) / (16 * sets);
  const bool staged_once = fours <= l.chunk_fours;
  auto stage = [&](long long first_four) {
    const long long dim0 = first_four * kFour;
    const int dims = (int)(min((long long)l.chunk_fours, fours - first_four) * kFour);
    for (int i = threadIdx.x; i < l.columns * dims; i += kScoreThreads) {
      const int c = i / dims, k = i % dims, q = c / Columns::kParts;
      unsigned short v = 0;
      if (q < nq && dim0 + k < p.d) v = Columns::part(x[(q0 + q) * p.query_stride + dim0 + k], c % Columns::kParts);
      xs[c * l.pitch + k] = v;
    }
  };
  if (staged_once) {
    stage(0);
    __syncthreads();
  }
  for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const long long row0 = tile * 16 * sets + 16 * set;
    // rows behind the last one are read as the last one and not written
    const long long ra = min(row0 + g, p.n - 1), rb = min(row0 + g + 8, p.n - 1);
    const unsigned char* ca = codes + ra * row_bytes;
    const unsigned char* cb = codes + rb * row_bytes;
    const __nv_bfloat16* sa = scales + ra * groups;
    const __nv_bfloat16* sb = scales + rb * groups;
    float total[kTiles][4];
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) total[i][j] = 0.0f;
    for (long long chunk = 0; chunk < fours; chunk += l.chunk_fours) {
      if (!staged_once) {
        __syncthreads();
        stage(chunk);
        __syncthreads();
      }
      const long long in_chunk = min((long long)l.chunk_fours, fours - chunk);
      const long long each = (in_chunk + l.split - 1) / l.split;
      const long long from = chunk + part * each, to = min(chunk + in_chunk, from + each);
      for (long long four = from; four < to; ++four) {
        const int m = (int)min(4ll, blocks - 4 * four);
        unsigned wa[4], wb[4];
        if (m == 4) {
          const uint4 a = __ldcs(reinterpret_cast<const uint4*>(ca + 64 * four + 16 * t));
          const uint4 b = __ldcs(reinterpret_cast<const uint4*>(cb + 64 * four + 16 * t));
          wa[0] = a.x, wa[1] = a.y, wa[2] = a.z, wa[3] = a.w;
          wb[0] = b.x, wb[1] = b.y, wb[2] = b.z, wb[3] = b.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            wa[j] = j < m ? *reinterpret_cast<const unsigned*>(ca + 64 * four + 4 * (t * m + j)) : 0x88888888u;
            wb[j] = j < m ? *reinterpret_cast<const unsigned*>(cb + 64 * four + 4 * (t * m + j)) : 0x88888888u;
          }
        }
        float sum[kTiles][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j >= m) break;
          const long long block = 4 * four + j;
          if (j == 0 || block % group_blocks == 0) {
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
              for (int k = 0; k < 4; ++k) sum[i][k] = 0.0f;
          }
          const unsigned a0[4] = {Pairs::template values<0>(wa[j]), Pairs::template values<0>(wb[j]),
                                  Pairs::template values<1>(wa[j]), Pairs::template values<1>(wb[j])};
          const unsigned a1[4] = {Pairs::template values<2>(wa[j]), Pairs::template values<2>(wb[j]),
                                  Pairs::template values<3>(wa[j]), Pairs::template values<3>(wb[j])};
          const unsigned short* column = xs + g * l.pitch + (four - chunk) * kFour + j * kBlock + 8 * t;
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            const uint4 b = *reinterpret_cast<const uint4*>(column + i * 8 * l.pitch);
            Pairs::mma(sum[i], a0, b.x, b.y);
            Pairs::mma(sum[i], a1, b.z, b.w);
          }
          if (j == m - 1 || (block + 1) % group_blocks == 0) {
            const float fa = __bfloat162float(sa[block / group_blocks]), fb = __bfloat162float(sb[block / group_blocks]);
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
              total[i][0] += fa * sum[i][0];
              total[i][1] += fa * sum[i][1];
              total[i][2] += fb * sum[i][2];
              total[i][3] += fb * sum[i][3];
            }
          }
        }
      }
    }
    // the shares and, of fp32 queries, the parts are added up in shared memory
    float* mine = sums + warp * l.columns * 17;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      mine[(8 * i + 2 * t) * 17 + g] = total[i][0];
      mine[(8 * i + 2 * t + 1) * 17 + g] = total[i][1];
      mine[(8 * i + 2 * t) * 17 + g + 8] = total[i][2];
      mine[(8 * i + 2 * t + 1) * 17 + g + 8] = total[i][3];
    }
    __syncthreads();
    const int rows = 16 * sets;
    for (int i = threadIdx.x; i < nq * rows; i += kScoreThreads) {
      const int q = i / rows, r = i % rows;
      const long long row = tile * rows + r;
      if (row >= p.n) continue;
      float y = 0.0f;
#pragma unroll
      for (int c = Columns::kParts - 1; c >= 0; --c)  // the small parts first
        for (int s = 0; s < l.split; ++s)
          y += sums[((r / 16) * l.split + s) * l.columns * 17 + (q * Columns::kParts + c) * 17 + r % 16];
      if (p.bias) y += p.bias[row];
      p.out[(q0 + q) * p.n + row] = y;
    }
    __syncthreads();
  }
}

template <class Columns, int kTiles>
cudaError_t scores_t(const Scores4Params& p, cudaStream_t stream) {
  constexpr int kSpace = 96 * 1024;  // of the queries in shared memory: two CTAs per SM
  ScoreLayout l;
  l.columns = 8 * kTiles;
  l.queries = l.columns / Columns::kParts;
  const long long fours = (p.d + kFour - 1) / kFour;
  const long long most = kSpace / (l.columns * 2 * kFour);
  l.chunk_fours = (int)(fours < most ? fours : most);
  // eight lanes read 16 bytes of two columns and four parts: half a row of banks from column to column
  l.pitch = l.chunk_fours * kFour + 32;
  const long long sets = (p.n + 15) / 16;
  l.split = 1;
  // rows for at least four CTAs per SM and every warp something to do
  while (l.split < kScoreWarps && 2 * l.split <= fours && sets * l.split < (long long)kSMs * 4 * kScoreWarps) l.split *= 2;
  const size_t smem = (size_t)l.columns * l.pitch * 2 + (size_t)kScoreWarps * l.columns * 17 * 4;
  cudaError_t e = cudaFuncSetAttribute(scores_kernel<Columns, kTiles>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  int per_sm = 0;
  e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, scores_kernel<Columns, kTiles>, kScoreThreads, smem);
  if (e != cudaSuccess) return e;
  const long long tiles = (sets + kScoreWarps / l.split - 1) / (kScoreWarps / l.split);
  const long long column_tiles = (p.nq + l.queries - 1) / l.queries;
  if (column_tiles > 65535) return cudaErrorInvalidValue;
  const long long room = (long long)kSMs * (per_sm > 0 ? per_sm : 1);
  const long long blocks = tiles < room ? tiles : room;
  scores_kernel<Columns, kTiles><<<dim3((unsigned)blocks, (unsigned)column_tiles), kScoreThreads, smem, stream>>>(p, l);
  return cudaGetLastError();
}

template <class Columns>
cudaError_t scores_columns(const Scores4Params& p, cudaStream_t stream) {
  const long long columns = p.nq * Columns::kParts;
  if (columns <= 8) return scores_t<Columns, 1>(p, stream);
  if (columns <= 16) return scores_t<Columns, 2>(p, stream);
  if (columns <= 24) return scores_t<Columns, 3>(p, stream);
  return scores_t<Columns, 4>(p, stream);
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
