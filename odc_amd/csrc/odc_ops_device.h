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

template <class T>
__device__ __forceinline__ float to_float(T x) { return (float)x; }
template <class T>
__device__ __forceinline__ T from_float(float x) { return (T)x; }  // to the nearest, ties to even

// The sum over the lanes of a wavefront, in every lane: pairs, then pairs of pairs.
template <class T>
__device__ __forceinline__ T wave_sum(T x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  return x;
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

// The item of a tile: the last one whose first tile is not behind it (items without elements have no tile).
template <class Launch>
__device__ __forceinline__ uint32_t item_of(const Launch& launch, uint32_t tile) {
  uint32_t low = 0, high = launch.n_items;
  while (high - low > 1) {
    const uint32_t mid = (low + high) / 2;
    if (launch.first_tile[mid] <= tile) low = mid; else high = mid;
  }
  return low;
}

}  // namespace odc_ops_device

#endif  // ODC_OPS_DEVICE_H_
