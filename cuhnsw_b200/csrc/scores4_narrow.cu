// Products of queries with 4-bit rows of up to 128 dimensions: one step of the matrix instruction's loop, so that what is done
// once per 32 rows counts.  The arithmetic is that of rows4.cu.  A warp has 32 rows at a time and nothing in common with the others
// but the queries in shared memory; the codes of its next rows are on their way in registers meanwhile, and the sums go from
// registers to where they belong, eight rows of four queries at a time.  Bound: instructions (some 250 for 32 rows of 50
// dimensions and 7 fp32 queries), behind them HBM bytes.  (7 fp32 queries and 1 183 514 rows of 50 dimensions 21 us, 3.4 TB/s;
// the kernel for longer rows 71.  One query and 1 000 000 rows of 128: 19 and 22.)
#include "scores4.cuh"

namespace hnsw {

namespace {

constexpr int kNarrowThreads = 256;
constexpr int kRowTiles = 2;                  // operands of 16 rows per warp
constexpr int kWarpRows = 16 * kRowTiles;
constexpr int kRowsPerLane = 2 * kRowTiles;   // rows g, g + 8, g + 16, g + 24
constexpr int kNarrowPitch = kFour + 32;      // values per column: half a row of banks from column to column

// M words of a row's part
template <int M>
__device__ __forceinline__ void load_words(const unsigned char* at, unsigned (&w)[M]) {
  if constexpr (M == 4) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(at));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (M == 2) {
    const uint2 v = __ldcs(reinterpret_cast<const uint2*>(at));
    w[0] = v.x, w[1] = v.y;
  } else {
#pragma unroll
    for (int j = 0; j < M; ++j) w[j] = __ldcs(reinterpret_cast<const unsigned*>(at) + j);
  }
}

// M: blocks of 32 dimensions; kGroup: blocks per scale, 4 for one scale per row.
template <class Columns, int kTiles, int M, int kGroup>
__global__ void __launch_bounds__(kNarrowThreads) narrow_kernel(const __grid_constant__ Scores4Params p, int queries,
                                                                int column_tiles) {
  using In = typename Columns::In;
  using Pairs = typename Columns::Pairs;
  constexpr int kOutTiles = kTiles / Columns::kParts, kScales = (M + kGroup - 1) / kGroup, kRowBytes = 16 * M;
  __shared__ __align__(16) unsigned short xs[8 * kTiles * kNarrowPitch];
  next_launch_may_start();
  wait_for_launch_before();
  const int warp = threadIdx.x >> 5, lane = lane_id(), g = lane >> 2, t = lane & 3;
  const long long q0 = (long long)(blockIdx.x % column_tiles) * queries;
  const int nq = (int)min((long long)queries, p.nq - q0);
  const unsigned rows = (unsigned)p.n, units = (rows + kWarpRows - 1) / kWarpRows;
  const unsigned step = gridDim.x / column_tiles * (kNarrowThreads / 32);
  unsigned unit = blockIdx.x / column_tiles * (kNarrowThreads / 32) + warp;
  // a warp's last rows are the table's last 32: some of them are another warp's as well, which writes the same
  const unsigned last_start = max(rows, (unsigned)kWarpRows) - kWarpRows;
  const int groups = (int)packed_groups_device(p.d, p.group);
  int row_at[kRowsPerLane];
#pragma unroll
  for (int i = 0; i < kRowsPerLane; ++i) row_at[i] = (int)min((unsigned)(g + 8 * i), rows - 1) * kRowBytes + 4 * t * M;
  const int scale_at = (int)min((unsigned)(g + 8 * t), rows - 1) * groups;  // lane t of a row's lanes loads row g + 8 * t's
  unsigned next_words[kRowsPerLane][M], next_scale[kScales];
  auto load = [&] {
    const long long row0 = min(unit * kWarpRows, last_start);
    const unsigned char* codes = static_cast<const unsigned char*>(p.codes) + row0 * kRowBytes;
    const unsigned short* scales = static_cast<const unsigned short*>(p.scales) + row0 * groups + scale_at;
#pragma unroll
    for (int i = 0; i < kRowsPerLane; ++i) load_words<M>(codes + row_at[i], next_words[i]);
#pragma unroll
    for (int i = 0; i < kScales; ++i) next_scale[i] = scales[i];
  };
  if (unit < units) load();
  const Pairs pairs;
  // the queries: a thread eight dimensions of one
  for (int i = threadIdx.x; i < nq * 4 * M; i += kNarrowThreads) {
    const int q = i / (4 * M), k = i % (4 * M) * 8;
    const In* src = static_cast<const In*>(p.queries) + (q0 + q) * p.query_stride;
#pragma unroll
    for (int c = 0; c < Columns::kParts; ++c) {
      unsigned w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const In low = k + 2 * j < p.d ? src[k + 2 * j] : from_f32<In>(0.0f);
        const In high = k + 2 * j + 1 < p.d ? src[k + 2 * j + 1] : from_f32<In>(0.0f);
        w[j] = (unsigned)Columns::part(low, c) | (unsigned)Columns::part(high, c) << 16;
      }
      *reinterpret_cast<uint4*>(xs + (c * nq + q) * kNarrowPitch + k) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __syncthreads();
  // lanes of columns that there are not read the last one's and throw the result away
  const unsigned short* column[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i)
    column[i] = xs + (Columns::kParts == 1 ? min(8 * i + g, nq - 1) : i * nq + min(g, nq - 1)) * kNarrowPitch + 8 * t;

  while (unit < units) {
    unsigned words[kRowsPerLane][M], scale[kScales];
#pragma unroll
    for (int i = 0; i < kRowsPerLane; ++i)
#pragma unroll
      for (int j = 0; j < M; ++j) words[i][j] = next_words[i][j];
#pragma unroll
    for (int i = 0; i < kScales; ++i) scale[i] = next_scale[i];
    const unsigned row0 = min(unit * kWarpRows, last_start);
    unit += step;
    if (unit < units) load();
    const bool whole = rows >= (unsigned)kWarpRows;
    float bias[kRowsPerLane];
#pragma unroll
    for (int i = 0; i < kRowsPerLane; ++i)
      bias[i] = p.bias && (whole || (unsigned)(g + 8 * i) < rows) ? p.bias[row0 + g + 8 * i] : 0.0f;
    float total[kRowTiles][kTiles][4];
#pragma unroll
    for (int s = 0; s < kScales; ++s) {
      float sum[kRowTiles][kTiles][4];
#pragma unroll
      for (int j = s * kGroup; j < M && j < (s + 1) * kGroup; ++j) {
        uint4 b[kTiles];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) b[i] = *reinterpret_cast<const uint4*>(column[i] + j * kBlock);
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r) {
          const unsigned wa = words[2 * r][j], wb = words[2 * r + 1][j];
          const unsigned a0[4] = {pairs.template values<0>(wa), pairs.template values<0>(wb),
                                  pairs.template values<1>(wa), pairs.template values<1>(wb)};
          const unsigned a1[4] = {pairs.template values<2>(wa), pairs.template values<2>(wb),
                                  pairs.template values<3>(wa), pairs.template values<3>(wb)};
#pragma unroll
          for (int i = 0; i < kTiles; ++i) Pairs::mma(sum[r][i], a0, b[i].x, b[i].y, j == s * kGroup);
#pragma unroll
          for (int i = 0; i < kTiles; ++i) Pairs::mma(sum[r][i], a1, b[i].z, b[i].w, false);
        }
      }
#pragma unroll
      for (int r = 0; r < kRowsPerLane; ++r) {
        const float f = bf16_low(__shfl_sync(FULL, scale[s], (lane & ~3) + r));
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float& y = total[r / 2][i][2 * (r % 2) + c];
            y = s == 0 ? f * sum[r / 2][i][2 * (r % 2) + c] : y + f * sum[r / 2][i][2 * (r % 2) + c];
          }
      }
    }
#pragma unroll
    for (int i = 0; i < kOutTiles; ++i) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int q = 8 * i + 2 * t + c;
        if (q < nq) {
          float* out = p.out + (q0 + q) * p.n + row0 + g;
#pragma unroll
          for (int r = 0; r < kRowsPerLane; ++r) {
            float y = total[r / 2][i * Columns::kParts][2 * (r % 2) + c];
            if constexpr (Columns::kParts == 3)
              y += total[r / 2][i * Columns::kParts + 1][2 * (r % 2) + c] +
                   total[r / 2][i * Columns::kParts + 2][2 * (r % 2) + c];
            if (whole || (unsigned)(g + 8 * r) < rows) out[8 * r] = y + bias[r];
          }
        }
      }
    }
  }
}

template <class Columns, int kTiles, int M, int kGroup>
cudaError_t narrow_t(const Scores4Params& p, int queries, cudaStream_t stream) {
  static std::atomic<int> per_sm{0};  // of the one architecture that this is compiled for
  int resident = per_sm.load(std::memory_order_relaxed);
  if (resident == 0) {
    const cudaError_t e =
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, narrow_kernel<Columns, kTiles, M, kGroup>, kNarrowThreads, 0);
    if (e != cudaSuccess) return e;
    if (resident < 1) resident = 1;
    per_sm.store(resident, std::memory_order_relaxed);
  }
  const int column_tiles = (int)((p.nq + queries - 1) / queries);
  const long long units = (p.n + kWarpRows - 1) / kWarpRows, wanted = (units + kNarrowThreads / 32 - 1) / (kNarrowThreads / 32);
  const long long room = ((long long)kSMs * resident + column_tiles - 1) / column_tiles;
  const long long blocks = wanted < room ? wanted : room;
  if (blocks * column_tiles > 0x7fffffffll) return cudaErrorInvalidValue;
  return launch_early(narrow_kernel<Columns, kTiles, M, kGroup>, dim3((unsigned)(blocks * column_tiles)), kNarrowThreads, 0,
                      stream, p, queries, column_tiles);
}

template <class Columns, int kTiles>
cudaError_t narrow_blocks(const Scores4Params& p, int queries, cudaStream_t stream) {
  const int m = (int)((p.d + kBlock - 1) / kBlock);
  const bool fine = p.group == kBlock, middle = p.group == 2 * kBlock;
  if (m == 1) return narrow_t<Columns, kTiles, 1, 4>(p, queries, stream);
  if (m == 2) return fine ? narrow_t<Columns, kTiles, 2, 1>(p, queries, stream) : narrow_t<Columns, kTiles, 2, 4>(p, queries, stream);
  if (m == 3)
    return fine     ? narrow_t<Columns, kTiles, 3, 1>(p, queries, stream)
           : middle ? narrow_t<Columns, kTiles, 3, 2>(p, queries, stream)
                    : narrow_t<Columns, kTiles, 3, 4>(p, queries, stream);
  return fine     ? narrow_t<Columns, kTiles, 4, 1>(p, queries, stream)
         : middle ? narrow_t<Columns, kTiles, 4, 2>(p, queries, stream)
                  : narrow_t<Columns, kTiles, 4, 4>(p, queries, stream);
}

template <class Columns>
cudaError_t narrow_columns(const Scores4Params& p, cudaStream_t stream) {
  // as many queries at a time as the operands have columns, in tiles of equal size
  const long long most = Columns::kParts == 1 ? 32 : 8, tiles = (p.nq + most - 1) / most;
  const int queries = (int)((p.nq + tiles - 1) / tiles);
  if constexpr (Columns::kParts == 3) {
    return narrow_blocks<Columns, 3>(p, queries, stream);
  } else {
    if (queries <= 8) return narrow_blocks<Columns, 1>(p, queries, stream);
    if (queries <= 16) return narrow_blocks<Columns, 2>(p, queries, stream);
    return narrow_blocks<Columns, 4>(p, queries, stream);
  }
}

}  // namespace

cudaError_t launch_scores4_narrow(const Scores4Params& p, cudaStream_t stream) {
  if (p.type == kF32) return narrow_columns<ColumnsF32>(p, stream);
  if (p.type == kF16) return narrow_columns<ColumnsF16>(p, stream);
  return narrow_columns<ColumnsBF16>(p, stream);
}

}  // namespace hnsw
