// What the kernels for products with 4-bit rows share: the format's units, how codes become values, queries columns.
#pragma once
#include "common.cuh"
#include "table_common.cuh"

namespace hnsw {

constexpr int kBlock = 32;             // dimensions of a block
constexpr int kFour = 4 * kBlock;      // of four blocks

__device__ __forceinline__ long long packed_groups_device(long long d, long long group) { return (d + group - 1) / group; }

// (bits & mask) | magic in one instruction: that takes one constant, the other one has to be in a register already
__device__ __forceinline__ unsigned and_or(unsigned bits, unsigned mask, unsigned magic) {
  unsigned r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(bits), "r"(mask), "r"(magic));
  return r;
}
__device__ __forceinline__ unsigned in_register(unsigned x) {
  unsigned r;
  asm volatile("mov.b32 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// c += a * b; `first`: c = a * b
#define MMA16816(types, c, a, b0, b1, first)                                                                         \
  if (first)                                                                                                         \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." types ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};" \
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])                                                             \
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));                                  \
  else                                                                                                               \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." types ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"  \
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])                                                             \
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1))

// Codes as values, in the way that is common for small whole numbers: their bits under the mantissa of a power of two, which is then
// taken away.
struct PairsF16 {
  unsigned magic = in_register(0x64006400u);  // 1024, the last bit of whose mantissa is one
  unsigned minus_low = in_register(0xe408e408u), sixteenth = in_register(0x2c002c00u), minus_high = in_register(0xd480d480u);
  // two codes of nibbles `pair` and `pair` + 4 as code - 8
  template <int Pair>
  __device__ __forceinline__ unsigned values(unsigned w) const {
    const unsigned u = Pair >= 2 ? w >> 8 : w;
    unsigned r;
    if (Pair % 2 == 0)  // 1024 + code - 1032
      asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(and_or(u, 0x000f000fu, magic)), "r"(minus_low));
    else  // (1024 + 16 * code) / 16 - 72
      asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(and_or(u, 0x00f000f0u, magic)), "r"(sixteenth), "r"(minus_high));
    return r;
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1, bool first) {
    MMA16816("f16.f16", c, a, b0, b1, first);
  }
};
struct PairsBF16 {
  unsigned magic = in_register(0x43004300u);  // 128
  unsigned minus = in_register(0xc308c308u), one = in_register(0x3f803f80u);
  template <int Pair>
  __device__ __forceinline__ unsigned values(unsigned w) const {
    unsigned r;  // 128 + code - 136
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(and_or(w >> (4 * Pair), 0x000f000fu, magic)), "r"(one), "r"(minus));
    return r;
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1, bool first) {
    MMA16816("bf16.bf16", c, a, b0, b1, first);
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
  static constexpr float kLargest = 0x1.fep127f;  // of bfloat16
  // x = high + middle + low: each part is what the ones before leave, rounded to 8 bits (below 2^-110 the last bits are lost)
  static __device__ __forceinline__ unsigned short part(float x, int which) {
    // (the largest numbers would round to infinity)
    const __nv_bfloat16 high = __float2bfloat16_rn(isfinite(x) ? fminf(fmaxf(x, -kLargest), kLargest) : x);
    if (which == 0) return __bfloat16_as_ushort(high);
    // (an infinity or NaN is all in the first part: its remainder would be a NaN)
    const float rest = isfinite(__bfloat162float(high)) ? x - __bfloat162float(high) : 0.0f;
    const __nv_bfloat16 middle = __float2bfloat16_rn(rest);
    return __bfloat16_as_ushort(which == 1 ? middle : __float2bfloat16_rn(rest - __bfloat162float(middle)));
  }
};

__device__ __forceinline__ float bf16_low(unsigned pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float bf16_high(unsigned pair) { return __uint_as_float(pair & 0xffff0000u); }

// The scales of a row for four blocks: bfloat16, one to four of them.  `at`: the first one; left: how many there are from there on.
template <int kGroup>
struct FourScales {
  unsigned low = 0, high = 0;
  __device__ __forceinline__ void load(const unsigned short* at, int left, bool wide) {
    if constexpr (kGroup == 4) {
      low = *at;
    } else if constexpr (kGroup == 2) {
      low = wide ? *reinterpret_cast<const unsigned*>(at) : (left > 0 ? at[0] : 0) | (left > 1 ? (unsigned)at[1] << 16 : 0);
    } else if (wide) {
      const uint2 both = *reinterpret_cast<const uint2*>(at);
      low = both.x;
      high = both.y;
    } else {
      low = at[0] | (left > 1 ? (unsigned)at[1] << 16 : 0);
      high = (left > 2 ? at[2] : 0) | (left > 3 ? (unsigned)at[3] << 16 : 0);
    }
  }
  __device__ __forceinline__ FourScales of_lane(int lane) const {
    FourScales r;
    r.low = __shfl_sync(FULL, low, lane);
    if (kGroup == 1) r.high = __shfl_sync(FULL, high, lane);
    return r;
  }
  __device__ __forceinline__ float get(int j) const {
    const unsigned pair = j < 2 ? low : high;
    return j % 2 == 0 ? bf16_low(pair) : bf16_high(pair);
  }
};

// Rows of up to 128 dimensions (scores4_narrow.cu)
cudaError_t launch_scores4_narrow(const Scores4Params& p, cudaStream_t stream);

}  // namespace hnsw
