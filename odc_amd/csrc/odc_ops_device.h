// odc_ops_device.h — what the kernels of libodc_ops.so share: types, sums over lanes and workgroups, the table
// of a list of tensors.
#ifndef ODC_OPS_DEVICE_H_
#define ODC_OPS_DEVICE_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "odc_ops.h"

namespace odc_ops_device {

typedef __bf16 bf16;
typedef _Float16 f16;

// `kernel` with what it takes; returns the launch's own status. (hipGetLastError() would also report what an earlier,
// unrelated HIP call of the same host thread left behind, and make a launch that runs look failed.)
template <class T>
struct Same { typedef T type; };
template <class... P>
int launch(void (*kernel)(P...), dim3 grid, uint32_t threads, void* stream, const typename Same<P>::type&... values) {
  void* args[] = {const_cast<void*>(static_cast<const void*>(&values))...};
  return (int)hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(threads), args, 0, static_cast<hipStream_t>(stream));
}

template <class T>
__device__ __forceinline__ float to_float(T x) { return (float)x; }
template <class T>
__device__ __forceinline__ T from_float(float x) { return (T)x; }  // to the nearest, ties to even

// 16 bytes of a type, as they are loaded and stored at any alignment that its elements have.
template <class T>
struct Vector {
  static constexpr int kElems = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
  typedef type unaligned __attribute__((aligned(sizeof(T))));
};

template <int kControl>
__device__ __forceinline__ float other_lane(float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), kControl, 0xf, 0xf, true));
}

// The sum over kLanes neighbouring lanes (a power of two up to 64), in every lane: by data-parallel primitives within 16
// lanes and by swaps of rows above, a few cycles each, where a shuffle through LDS takes over 50. Neighbours, pairs,
// ...: the order is the same for all lanes.
template <int kLanes>
__device__ __forceinline__ float sum_lanes(float x) {
  if constexpr (kLanes > 1) x += other_lane<0xB1>(x);   // quad_perm 1 0 3 2
  if constexpr (kLanes > 2) x += other_lane<0x4E>(x);   // quad_perm 2 3 0 1
  if constexpr (kLanes > 4) x += other_lane<0x141>(x);  // mirrored within 8
  if constexpr (kLanes > 8) x += other_lane<0x140>(x);  // mirrored within 16
  if constexpr (kLanes > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (kLanes > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return x;
}

// The sum over the lanes of a wavefront, in every lane.
__device__ __forceinline__ float wave_sum(float x) { return sum_lanes<64>(x); }
// In 64 bits the same, a half of the bits at a time.
__device__ __forceinline__ double of_halves(uint32_t low, uint32_t high) { return __longlong_as_double((long long)((uint64_t)high << 32 | low)); }
template <int kControl>
__device__ __forceinline__ double other_lane(double x) {
  const uint64_t bits = (uint64_t)__double_as_longlong(x);
  return of_halves(__builtin_amdgcn_update_dpp(0, (uint32_t)bits, kControl, 0xf, 0xf, true),
                   __builtin_amdgcn_update_dpp(0, (uint32_t)(bits >> 32), kControl, 0xf, 0xf, true));
}
__device__ __forceinline__ double wave_sum(double x) {
  x += other_lane<0xB1>(x);
  x += other_lane<0x4E>(x);
  x += other_lane<0x141>(x);
  x += other_lane<0x140>(x);
  uint64_t bits = (uint64_t)__double_as_longlong(x);
  auto low = __builtin_amdgcn_permlane16_swap((uint32_t)bits, (uint32_t)bits, false, false);
  auto high = __builtin_amdgcn_permlane16_swap((uint32_t)(bits >> 32), (uint32_t)(bits >> 32), false, false);
  x = of_halves(low[0], high[0]) + of_halves(low[1], high[1]);
  bits = (uint64_t)__double_as_longlong(x);
  low = __builtin_amdgcn_permlane32_swap((uint32_t)bits, (uint32_t)bits, false, false);
  high = __builtin_amdgcn_permlane32_swap((uint32_t)(bits >> 32), (uint32_t)(bits >> 32), false, false);
  return of_halves(low[0], high[0]) + of_halves(low[1], high[1]);
}

// The sum over a workgroup of kThreads, in every thread. `scratch` holds kThreads / 64 values.
template <int kThreads, class T>
__device__ __forceinline__ T block_sum(T x, T* scratch) {
  constexpr int kWaves = kThreads / 64;
  x = wave_sum(x);
  if constexpr (kWaves > 1) {
    __syncthreads();  // the last sum's readers are done
    if (threadIdx.x % 64 == 0) scratch[threadIdx.x / 64] = x;
    __syncthreads();
    x = scratch[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) x += scratch[w];
  }
  return x;
}

// The item of a tile: the last one whose first tile is not behind it (items without elements have no tile). By scalar
// loads, each of which waits for the one before.
template <class Launch>
__device__ __forceinline__ uint32_t item_of(const Launch& launch, uint32_t tile) {
  uint32_t low = 0, high = launch.n_items;
  while (high - low > 1) {
    const uint32_t mid = (low + high) / 2;
    if (launch.first_tile[mid] <= tile) low = mid; else high = mid;
  }
  return low;
}

// The same for a long table: every lane looks at items of its own, all at once. (The squared norm of 300 small tensors
// took 25 us in two launches by the search above, 13 in one by this; an AdamW step over nine, whose table is short,
// 142 and 150.)
template <class Launch>
__device__ __forceinline__ uint32_t item_of_many(const Launch& launch, uint32_t tile) {
  constexpr uint32_t kItems = sizeof(launch.first_tile) / sizeof(uint32_t) - 1;
  const uint32_t lane = threadIdx.x % 64;
  uint32_t begun = 0;
#pragma unroll
  for (uint32_t i = 0; i < kItems; i += 64) {
    const uint32_t k = i + lane;
    begun += __popcll(__ballot(k < launch.n_items && launch.first_tile[k < kItems ? k : 0] <= tile));
  }
  return __builtin_amdgcn_readfirstlane(begun) - 1;
}

}  // namespace odc_ops_device

#endif  // ODC_OPS_DEVICE_H_
