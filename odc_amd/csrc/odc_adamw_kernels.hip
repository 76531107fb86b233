// odc_adamw_kernels.hip — the squared norm and the AdamW step of many tensors for gfx950.
#include "odc_ops_device.h"
#include "odc_ops_launch.h"

namespace odc_ops_device {
namespace {

using namespace odc_ops_launch;

// ---- squared norm ---------------------------------------------------------------------------------
template <class T>
__global__ __launch_bounds__(256) void squared_norm_kernel(SquaredNormLaunch launch, double* partials) {
  __shared__ double scratch[4];
  float sum = 0;
  for (uint32_t tile = blockIdx.x; tile < launch.n_tiles; tile += gridDim.x) {
    const uint32_t k = item_of(launch, tile);
    const T* data = static_cast<const T*>(launch.items[k].data);
    const uint64_t first = (uint64_t)(tile - launch.first_tile[k]) * kNormTile;
    const uint64_t end = first + kNormTile < launch.items[k].elems ? first + kNormTile : launch.items[k].elems;
    for (uint64_t i = first + threadIdx.x; i < end; i += 256) {
      const float x = to_float(data[i]);
      sum += x * x;
    }
  }
  const double all = block_sum<256>((double)sum, scratch);
  if (threadIdx.x == 0) partials[blockIdx.x] = all;
}

__global__ __launch_bounds__(256) void squared_norm_total_kernel(const double* partials, uint32_t n, float* result) {
  __shared__ double scratch[4];
  double sum = 0;
  for (uint32_t i = threadIdx.x; i < n; i += 256) sum += partials[i];
  sum = block_sum<256>(sum, scratch);
  if (threadIdx.x == 0) *result = (float)sum;
}

// ---- AdamW ----------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t mix(uint32_t x) {
  x = (x ^ (x >> 16)) * 0xB7E15163u;
  x = (x ^ (x >> 15)) * 0x9E3779B1u;
  return x ^ (x >> 16);
}

// The factor of the gradients. A norm that is not a number makes it not a number.
__device__ __forceinline__ float factor_of(const AdamwLaunch& launch) {
  if (!launch.squared_norm) return launch.grad_scale;
  const float c = launch.max_norm / (launch.grad_scale * sqrtf(*launch.squared_norm) + 1e-6f);
  return launch.grad_scale * (c > 1.0f ? 1.0f : c);
}

struct Moments {
  float m, v, root;
};

__device__ __forceinline__ Moments next_moments(const AdamwLaunch& launch, float g, float m, float v) {
  Moments out;
  out.m = m * launch.beta1 + g * launch.one_minus_beta1;
  out.v = v * launch.beta2 + g * g * launch.one_minus_beta2;
  out.root = sqrtf(out.v);
  return out;
}

__device__ __forceinline__ float next_param(const AdamwLaunch& launch, float p, const Moments& s) {
  return p * launch.decay - launch.step_size * (s.m / (s.root * launch.root_scale + launch.eps));
}

// The biased exponent of a block's scale from its largest value: the smallest power of two that keeps it
// within 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t scale_of(float largest) {
  const int k = (int)((__float_as_uint(largest) + 0x1FFFFFu) >> 23) - 8;
  return k < 10 ? 10u : (uint32_t)k;
}

// The e4m3 value beside |x| / scale that the 16 bits of `chance` choose, as code; x's sign with it. kSquares:
// the expectation of the square is kept.
template <bool kSquares>
__device__ __forceinline__ uint32_t code_of(float x, uint32_t scale, uint32_t chance) {
  if (!(fabsf(x) < INFINITY)) return 0x7F;
  float size = fabsf(x) * __uint_as_float((254u - scale) << 23);
  if (kSquares && size > 0) size = fmaxf(size, 0x1p-9f);
  const float step = __uint_as_float(__float_as_uint(fmaxf(size, 0x1p-6f)) & 0x7F800000u) * 0.125f;
  const float below = floorf(size / step) * step;
  float share = size - below, whole = step;
  if (kSquares) {
    share *= size + below;
    whole *= below + below + step;
  }
  const float chosen = ((float)chance + 0.5f) * whole < share * 65536.0f ? below + step : below;
  const uint32_t pair = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(copysignf(chosen, x), 0.0f, 0, false);
  return pair & 0xFF;
}

__device__ __forceinline__ float value_of(uint32_t code, uint32_t scale) {
  return __builtin_amdgcn_cvt_f32_fp8((int)code, 0) * __uint_as_float(scale << 23);
}

template <class P, class G, class C>
__global__ __launch_bounds__(kAdamwThreads) void adamw_kernel(AdamwLaunch launch) {
  const uint32_t k = item_of(launch, blockIdx.x);
  const odc_adamw_item& it = launch.items[k];
  const float factor = factor_of(launch);
  const uint64_t first = (uint64_t)(blockIdx.x - launch.first_tile[k]) * kAdamwTile;
  for (uint32_t j = threadIdx.x; j < kAdamwTile; j += kAdamwThreads) {
    const uint64_t i = first + j;
    if (i >= it.elems) break;
    const float g = to_float(static_cast<const G*>(it.grad)[i]) * factor;
    float* m = static_cast<float*>(it.exp_avg) + i;
    float* v = static_cast<float*>(it.exp_avg_sq) + i;
    P* param = static_cast<P*>(it.param) + i;
    const Moments s = next_moments(launch, g, *m, *v);
    *m = s.m;
    *v = s.v;
    const float p = next_param(launch, to_float(*param), s);
    if (sizeof(P) == 2 && launch.stochastic) {
      const uint64_t n = i;
      const uint32_t word = mix((uint32_t)n + (uint32_t)(n >> 32) * 0x632BE5ABu + mix(launch.seed + (launch.first_item + k) * 0x9E3779B1u));
      uint32_t bits = __float_as_uint(p);
      if (fabsf(p) < INFINITY) bits = (bits + (mix(word ^ 0x5BF03635u) & 0xFFFFu)) & 0xFFFF0000u;
      *param = from_float<P>(__uint_as_float(bits));
    } else {
      *param = from_float<P>(p);
    }
    if (it.copy) static_cast<C*>(it.copy)[i] = from_float<C>(p);
  }
}

// A block of 32 elements is half a wavefront, whose lanes all come along.
template <class P, class G, class C>
__global__ __launch_bounds__(kAdamwThreads) void adamw8_kernel(AdamwLaunch launch) {
  const uint32_t k = item_of(launch, blockIdx.x);
  const odc_adamw_item& it = launch.items[k];
  const float factor = factor_of(launch);
  const uint32_t key = mix(launch.seed + (launch.first_item + k) * 0x9E3779B1u);
  const uint64_t first = (uint64_t)(blockIdx.x - launch.first_tile[k]) * kAdamwTile;
  uint8_t* codes_m = static_cast<uint8_t*>(it.exp_avg);
  uint8_t* codes_v = static_cast<uint8_t*>(it.exp_avg_sq);
  uint8_t* scales_m = static_cast<uint8_t*>(it.exp_avg_scale);
  uint8_t* scales_v = static_cast<uint8_t*>(it.exp_avg_sq_scale);
  for (uint32_t j = threadIdx.x; j < kAdamwTile; j += kAdamwThreads) {
    const uint64_t i = first + j, block = i / kBlock;
    const bool mine = i < it.elems;
    Moments s = {0, 0, 0};
    P* param = static_cast<P*>(it.param) + i;
    if (mine) {
      const float g = to_float(static_cast<const G*>(it.grad)[i]) * factor;
      const float root = value_of(codes_v[i], scales_v[block]);
      s = next_moments(launch, g, value_of(codes_m[i], scales_m[block]), root * root);
    }
    float top_m = fabsf(s.m) < INFINITY ? fabsf(s.m) : 0, top_v = s.root < INFINITY ? s.root : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      top_m = fmaxf(top_m, __shfl_xor(top_m, d));
      top_v = fmaxf(top_v, __shfl_xor(top_v, d));
    }
    if (!mine) continue;
    const uint32_t scale_m = scale_of(top_m), scale_v = scale_of(top_v);
    const uint32_t word = mix((uint32_t)i + (uint32_t)(i >> 32) * 0x632BE5ABu + key);
    codes_m[i] = (uint8_t)code_of<false>(s.m, scale_m, word & 0xFFFFu);
    codes_v[i] = (uint8_t)code_of<true>(s.root, scale_v, word >> 16);
    if (i % kBlock == 0) {
      scales_m[block] = (uint8_t)scale_m;
      scales_v[block] = (uint8_t)scale_v;
    }
    const float p = next_param(launch, to_float(*param), s);
    if (sizeof(P) == 2 && launch.stochastic) {
      uint32_t bits = __float_as_uint(p);
      if (fabsf(p) < INFINITY) bits = (bits + (mix(word ^ 0x5BF03635u) & 0xFFFFu)) & 0xFFFF0000u;
      *param = from_float<P>(__uint_as_float(bits));
    } else {
      *param = from_float<P>(p);
    }
    if (it.copy) static_cast<C*>(it.copy)[i] = from_float<C>(p);
  }
}

template <class T>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t* codes, const uint8_t* scales, T* values, uint64_t elems) {
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < elems; i += (uint64_t)gridDim.x * 256)
    values[i] = from_float<T>(value_of(codes[i], scales[i / kBlock]));
}

template <class Body>
int with_type(int32_t dtype, Body body) {
  return dtype == ODC_OPS_F32 ? body(float()) : dtype == ODC_OPS_BF16 ? body(bf16()) : body(f16());
}

}  // namespace

int launch_squared_norm(int32_t dtype, const SquaredNormLaunch& launch, uint32_t blocks, double* partials, void* stream) {
  return with_type(dtype, [&](auto t) {
    squared_norm_kernel<decltype(t)><<<blocks, 256, 0, (hipStream_t)stream>>>(launch, partials);
    return (int)hipGetLastError();
  });
}

int launch_squared_norm_total(const double* partials, uint32_t n, float* result, void* stream) {
  squared_norm_total_kernel<<<1, 256, 0, (hipStream_t)stream>>>(partials, n, result);
  return (int)hipGetLastError();
}

int launch_adamw(int32_t param, int32_t grad, int32_t copy, int32_t state_bits, const AdamwLaunch& launch, void* stream) {
  return with_type(grad, [&](auto g) {
    const auto with_param = [&](auto p, auto c) {
      if (state_bits == 8) adamw8_kernel<decltype(p), decltype(g), decltype(c)><<<launch.n_tiles, kAdamwThreads, 0, (hipStream_t)stream>>>(launch);
      else adamw_kernel<decltype(p), decltype(g), decltype(c)><<<launch.n_tiles, kAdamwThreads, 0, (hipStream_t)stream>>>(launch);
      return (int)hipGetLastError();
    };
    if (param == ODC_OPS_BF16) return with_param(bf16(), bf16());
    return copy == ODC_OPS_F16 ? with_param(float(), f16()) : with_param(float(), bf16());
  });
}

int launch_dequantize(const void* codes, const void* scales, void* values, uint64_t elems, int32_t dtype, void* stream) {
  return with_type(dtype, [&](auto t) {
    const uint64_t blocks = (elems + 255) / 256;
    dequantize_kernel<decltype(t)><<<(uint32_t)(blocks < 65536 ? blocks : 65536), 256, 0, (hipStream_t)stream>>>(
        static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), static_cast<decltype(t)*>(values), elems);
    return (int)hipGetLastError();
  });
}

}  // namespace odc_ops_device
