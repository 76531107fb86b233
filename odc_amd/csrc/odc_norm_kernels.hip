// odc_norm_kernels.hip — layer norm forward and backward for gfx950.
#include "odc_ops_device.h"
#include "odc_ops_launch.h"

namespace odc_ops_device {
namespace {

using namespace odc_ops_launch;

// One workgroup per row, three passes over it (the second and third find it in the caches): the mean, the
// variance about that mean, the output.
template <class T, class W>
__global__ __launch_bounds__(kNormThreads) void norm_forward_kernel(odc_norm_forward c) {
  __shared__ float scratch[kNormThreads / 64];
  const W* weight = static_cast<const W*>(c.weight);
  const W* bias = static_cast<const W*>(c.bias);
  for (uint64_t row = blockIdx.x; row < c.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(c.input) + row * c.input_stride;
    const T* r = c.residual ? static_cast<const T*>(c.residual) + row * c.residual_stride : nullptr;
    T* y = static_cast<T*>(c.output) + row * c.width;
    T* total = r ? static_cast<T*>(c.total) + row * c.width : nullptr;
    float sum = 0;
    for (uint64_t i = threadIdx.x; i < c.width; i += kNormThreads) {
      float v = to_float(x[i]);
      if (r) {
        const T t = from_float<T>(v + to_float(r[i]));
        total[i] = t;
        v = to_float(t);
      }
      sum += v;
    }
    const T* z = r ? total : x;  // a thread reads what it wrote itself
    const float mean = block_sum<kNormThreads>(sum, scratch) / (float)c.width;
    float squares = 0;
    for (uint64_t i = threadIdx.x; i < c.width; i += kNormThreads) {
      const float d = to_float(z[i]) - mean;
      squares += d * d;
    }
    const float rstd = 1.0f / sqrtf(block_sum<kNormThreads>(squares, scratch) / (float)c.width + c.eps);
    for (uint64_t i = threadIdx.x; i < c.width; i += kNormThreads) {
      float v = (to_float(z[i]) - mean) * rstd;
      if (weight) v *= to_float(weight[i]);
      if (bias) v += to_float(bias[i]);
      y[i] = from_float<T>(v);
    }
    if (threadIdx.x == 0) {
      if (c.mean) c.mean[row] = mean;
      if (c.rstd) c.rstd[row] = rstd;
    }
  }
}

template <class T, class W>
__global__ __launch_bounds__(kNormThreads) void norm_backward_rows_kernel(odc_norm_backward c) {
  __shared__ float scratch[kNormThreads / 64];
  const W* weight = static_cast<const W*>(c.weight);
  for (uint64_t row = blockIdx.x; row < c.rows; row += gridDim.x) {
    const T* dy = static_cast<const T*>(c.grad_output) + row * c.grad_output_stride;
    const T* x = static_cast<const T*>(c.normalised) + row * c.normalised_stride;
    const T* dt = c.grad_total ? static_cast<const T*>(c.grad_total) + row * c.grad_total_stride : nullptr;
    T* dx = static_cast<T*>(c.grad_input) + row * c.width;
    const float mean = c.mean[row], rstd = c.rstd[row];
    float sum = 0, dot = 0;
    for (uint64_t i = threadIdx.x; i < c.width; i += kNormThreads) {
      const float h = to_float(dy[i]) * (weight ? to_float(weight[i]) : 1.0f);
      sum += h;
      dot += h * ((to_float(x[i]) - mean) * rstd);
    }
    sum = block_sum<kNormThreads>(sum, scratch) / (float)c.width;
    dot = block_sum<kNormThreads>(dot, scratch) / (float)c.width;
    for (uint64_t i = threadIdx.x; i < c.width; i += kNormThreads) {
      const float h = to_float(dy[i]) * (weight ? to_float(weight[i]) : 1.0f);
      const float z = (to_float(x[i]) - mean) * rstd;
      float d = rstd * (h - sum - z * dot);
      if (dt) d += to_float(dt[i]);
      dx[i] = from_float<T>(d);
    }
  }
}

// Workgroup (tile of columns, group of rows): the sums over the group's rows. Wavefront w takes every fourth row.
template <class T>
__global__ __launch_bounds__(kNormThreads) void norm_backward_columns_kernel(odc_norm_backward c, uint64_t rows_per_group) {
  constexpr int kWaves = kNormThreads / 64;
  __shared__ float scratch[2][kWaves][64];
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const uint64_t column = (uint64_t)blockIdx.x * kColumnTile + lane;
  const uint64_t first = blockIdx.y * rows_per_group;
  const uint64_t end = first + rows_per_group < c.rows ? first + rows_per_group : c.rows;
  float dw = 0, db = 0;
  if (column < c.width) {
    for (uint64_t row = first + wave; row < end; row += kWaves) {
      const float dy = to_float(static_cast<const T*>(c.grad_output)[row * c.grad_output_stride + column]);
      const float x = to_float(static_cast<const T*>(c.normalised)[row * c.normalised_stride + column]);
      dw += dy * ((x - c.mean[row]) * c.rstd[row]);
      db += dy;
    }
  }
  scratch[0][wave][lane] = dw;
  scratch[1][wave][lane] = db;
  __syncthreads();
  if (wave < 2 && column < c.width) {
    float sum = scratch[wave][0][lane];
    for (int w = 1; w < kWaves; ++w) sum += scratch[wave][w][lane];
    static_cast<float*>(c.workspace)[(2 * (uint64_t)blockIdx.y + wave) * c.width + column] = sum;
  }
}

template <class W>
__global__ __launch_bounds__(kNormThreads) void norm_backward_groups_kernel(odc_norm_backward c, uint32_t groups) {
  const uint64_t at = (uint64_t)blockIdx.x * kNormThreads + threadIdx.x;  // of [2][width]
  if (at >= 2 * c.width) return;
  float sum = 0;
  for (uint32_t g = 0; g < groups; ++g) sum += static_cast<const float*>(c.workspace)[g * 2 * c.width + at];
  W* out = static_cast<W*>(at < c.width ? c.grad_weight : c.grad_bias);
  if (out) out[at % c.width] = from_float<W>(sum);
}

// Calls body with a value of the element types' own.
template <class Body>
int with_types(int32_t dtype, int32_t weight_dtype, Body body) {
  if (dtype == ODC_OPS_F32) return body(float(), float());
  if (dtype == ODC_OPS_BF16) return weight_dtype == ODC_OPS_F32 ? body(bf16(), float()) : body(bf16(), bf16());
  return weight_dtype == ODC_OPS_F32 ? body(f16(), float()) : body(f16(), f16());
}

}  // namespace

int launch_norm_forward(const odc_norm_forward& call, const NormForwardPlan& plan, void* stream) {
  return with_types(call.dtype, call.weight_dtype, [&](auto t, auto w) {
    norm_forward_kernel<decltype(t), decltype(w)><<<plan.blocks, kNormThreads, 0, (hipStream_t)stream>>>(call);
    return (int)hipGetLastError();
  });
}

int launch_norm_backward(const odc_norm_backward& call, const NormBackwardPlan& plan, void* stream) {
  return with_types(call.dtype, call.weight_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    hipStream_t s = (hipStream_t)stream;
    if (call.rows && call.grad_input) norm_backward_rows_kernel<T, W><<<plan.row_blocks, kNormThreads, 0, s>>>(call);
    if (call.grad_weight || call.grad_bias) {
      const uint32_t tiles = (uint32_t)((call.width + kColumnTile - 1) / kColumnTile);
      if (plan.groups) norm_backward_columns_kernel<T><<<dim3(tiles, plan.groups), kNormThreads, 0, s>>>(call, plan.rows_per_group);
      const uint32_t blocks = (uint32_t)((2 * call.width + kNormThreads - 1) / kNormThreads);
      norm_backward_groups_kernel<W><<<blocks, kNormThreads, 0, s>>>(call, plan.groups);
    }
    return (int)hipGetLastError();
  });
}

const char* error_string(int code) { return hipGetErrorString((hipError_t)code); }

}  // namespace odc_ops_device
