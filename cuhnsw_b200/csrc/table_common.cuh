// What the kernels over a table of embeddings share: element types and vectors of them.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "table.h"

namespace hnsw {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N values that are loaded and stored as one word of up to 16 bytes
template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

template <int Bytes>
struct WordOf;
template <>
struct WordOf<16> { using type = uint4; };
template <>
struct WordOf<8> { using type = uint2; };
template <>
struct WordOf<4> { using type = unsigned; };
template <>
struct WordOf<2> { using type = unsigned short; };

template <class T, int N>
__device__ __forceinline__ Vec<T, N> load_vec(const T* p) {
  using W = typename WordOf<sizeof(T) * N>::type;
  const W w = *reinterpret_cast<const W*>(p);
  return *reinterpret_cast<const Vec<T, N>*>(&w);
}
template <class T, int N>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, N>& v) {
  using W = typename WordOf<sizeof(T) * N>::type;
  *reinterpret_cast<W*>(p) = *reinterpret_cast<const W*>(&v);
}

// N values of T in words of 16 bytes, or in one of less
template <class T, int N>
__device__ __forceinline__ void load_many(const T* p, T (&v)[N]) {
  constexpr int kEach = N * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
  for (int i = 0; i < N; i += kEach) {
    const Vec<T, kEach> w = load_vec<T, kEach>(p + i);
#pragma unroll
    for (int j = 0; j < kEach; ++j) v[i + j] = w.v[j];
  }
}
template <class T, int N>
__device__ __forceinline__ void store_many(T* p, const T (&v)[N]) {
  constexpr int kEach = N * (int)sizeof(T) > 16 ? 16 / (int)sizeof(T) : N;
#pragma unroll
  for (int i = 0; i < N; i += kEach) {
    Vec<T, kEach> w;
#pragma unroll
    for (int j = 0; j < kEach; ++j) w.v[j] = v[i + j];
    store_vec<T, kEach>(p + i, w);
  }
}

// The widest word, 16 bytes at most, that every address and length in `bits` (their bitwise or) is a multiple of.
inline int word_bytes(unsigned long long bits) {
  for (int w = 16; w > 1; w >>= 1)
    if (bits % w == 0) return w;
  return 1;
}

inline int next_pow2(long long x, int at_most) {
  int p = 1;
  while (p < x && p < at_most) p <<= 1;
  return p;
}

constexpr int kSMs = 148;

// Lets a kernel have as much shared memory as there is; asked for once per device.
template <auto kKernel>
cudaError_t allow_smem() {
  constexpr int kMost = 227 * 1024 - 2048;  // and what it declares statically
  static std::atomic<bool> done[64];
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess || (device < 64 && done[device].load(std::memory_order_relaxed))) return e;
  e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
  if (e == cudaSuccess && device < 64) done[device].store(true, std::memory_order_relaxed);
  return e;
}

// A launch that may be set up while the one before it on the stream still runs: its kernel calls wait_for_launch_before() ahead of
// everything that it reads or writes in common with what came before, and next_launch_may_start() as soon as the one after it may be
// set up.  Saves one to two microseconds a launch.  Such a kernel is alive while its inputs may still be written, so it reads them by
// ordinary loads: read-only ones (__ldg, ld.global.nc) are for what does not change as long as a kernel lives.
__device__ __forceinline__ void wait_for_launch_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void next_launch_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class... Params, class... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3((unsigned)threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
}

}  // namespace hnsw
