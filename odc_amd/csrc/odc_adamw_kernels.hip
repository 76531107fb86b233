// odc_adamw_kernels.hip — the squared norm and the AdamW step of many tensors for gfx950.
//
// The formulas are in include/odc_ops.h. All of it is one pass over memory: 28 bytes for an element of an fp32 step, 16.1 with states
// in 8 bits, 10.1 with bf16 parameters and gradients beside those. HBM bounds all but the last, which its 88 instructions do.
// Measured: fp32 4.33 to 4.50 ms over 1.0 G elements (6.2 to 6.5 TB/s), with bf16 parameters and gradients 333 us over 100 M (6.6 TB/s
// at 22 bytes); 8 bits 67 to 70 us over 27.3 M (6.3 to 6.6 TB/s); bf16 with 8 bits 31 us over 11.2 M (3.6 TB/s); the squared norm
// 287 us over 1.0 G bf16 elements (7.0 TB/s), 7.2 us over 300 small tensors.
#include <type_traits>

#include "odc_ops_device.h"
#include "odc_ops_launch.h"

namespace odc_ops_device {
namespace {

using namespace odc_ops_launch;

// ---- squared norm ---------------------------------------------------------------------------------
// Every lane adds up the 32 squares that it has of a tile in fp32, the tiles in 64 bits.
template <class T, bool kStream>
__global__ __launch_bounds__(256) void squared_norm_kernel(SquaredNormLaunch launch, double* partials) {
  constexpr uint32_t kElems = Vector<T>::kElems, kSteps = kNormTile / (256 * kElems);
  __shared__ double scratch[4];
  double total = 0;
  for (uint32_t tile = blockIdx.x; tile < launch.n_tiles; tile += gridDim.x) {
    const uint32_t k = item_of_many(launch, tile);
    const uint64_t place = launch.places[k];
    const uint32_t tile_of_item = tile - launch.first_tile[k];
    const uint32_t left = tile + 1 < launch.first_tile[k + 1] ? kNormTile : (uint32_t)(place & 0xFFFF);
    const T* data = reinterpret_cast<const T*>(place >> 16) + (uint64_t)tile_of_item * kNormTile;
    float sum[kElems] = {};
    if (left >= kNormTile) {
      typename Vector<T>::type x[kSteps];
#pragma unroll
      for (uint32_t s = 0; s < kSteps; ++s) {
        const auto* p = reinterpret_cast<const typename Vector<T>::unaligned*>(data + (s * 256 + threadIdx.x) * kElems);
        if constexpr (kStream) x[s] = __builtin_nontemporal_load(p);
        else x[s] = *p;
      }
#pragma unroll
      for (uint32_t s = 0; s < kSteps; ++s)
#pragma unroll
        for (uint32_t e = 0; e < kElems; ++e) sum[e] += to_float(x[s][e]) * to_float(x[s][e]);
    } else {
      for (uint32_t i = threadIdx.x * kElems; i < left; i += 256 * kElems) {
        if (i + kElems <= left) {
          const typename Vector<T>::type x = *reinterpret_cast<const typename Vector<T>::unaligned*>(data + i);
#pragma unroll
          for (uint32_t e = 0; e < kElems; ++e) sum[e] += to_float(x[e]) * to_float(x[e]);
        } else {
#pragma unroll
          for (uint32_t e = 0; e < kElems; ++e) {
            const float x = i + e < left ? to_float(data[i + e]) : 0.0f;
            sum[e] += x * x;
          }
        }
      }
    }
#pragma unroll
    for (uint32_t width = kElems / 2; width; width /= 2)
#pragma unroll
      for (uint32_t e = 0; e < width; ++e) sum[e] += sum[e + width];
    total += sum[0];
  }
  total = block_sum<256>(total, scratch);
  if (threadIdx.x == 0) partials[blockIdx.x] = total;
}

__global__ __launch_bounds__(256) void squared_norm_total_kernel(const double* partials, uint32_t n, float* result) {
  __shared__ double scratch[4];
  double sum = 0;
#pragma unroll 8
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

// The square root and the reciprocal of the hardware (1 ulp each), which take a subnormal number for zero. Only a v can be
// one here: its root goes by root_of.
__device__ __forceinline__ float fast_sqrt(float x) { return __builtin_amdgcn_sqrtf(x); }
__device__ __forceinline__ float fast_reciprocal(float x) { return __builtin_amdgcn_rcpf(x); }

__device__ __forceinline__ float root_of(float v) {
  const bool small = v < 0x1p-96f;
  const float r = fast_sqrt(small ? v * 0x1p32f : v);
  return small ? r * 0x1p-16f : r;
}

// The factor of the gradients, one number for all of them: its root and its division are rounded to the nearest. A norm that is
// not a number makes it not a number.
__device__ __forceinline__ float factor_of(const AdamwLaunch& launch) {
  if (!launch.squared_norm) return launch.grad_scale;
  const float c = launch.max_norm / (launch.grad_scale * sqrtf(*launch.squared_norm) + 1e-6f);
  return launch.grad_scale * (c > 1.0f ? 1.0f : c);
}

// Four neighbouring elements, as a lane works on them: 16 bytes in fp32, so that a wavefront's accesses to every
// list are whole lines. kStream: nontemporal. Only the first n of the four exist.
template <class T>
struct Four {
  typedef T type __attribute__((ext_vector_type(4)));
  typedef type unaligned __attribute__((aligned(sizeof(T))));
  type v;

  template <bool kStream>
  __device__ __forceinline__ void load(const T* p, uint32_t n) {
    if (n == 4) {
      const auto* q = reinterpret_cast<const unaligned*>(p);
      if constexpr (kStream) v = __builtin_nontemporal_load(q);
      else v = *q;
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) v[e] = e < n ? p[e] : (T)0;
    }
  }
  template <bool kStream>
  __device__ __forceinline__ void store(T* p, uint32_t n) const {
    if (n == 4) {
      auto* q = reinterpret_cast<unaligned*>(p);
      if constexpr (kStream) __builtin_nontemporal_store((unaligned)v, q);
      else *q = v;
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 3; ++e)
        if (e < n) p[e] = v[e];
    }
  }
};

// The roots of four values. Small ones are rare: a wavefront without any takes the instruction as it is.
__device__ __forceinline__ void roots_of(const float (&v)[4], float (&root)[4]) {
  const float least = fminf(fminf(v[0], v[1]), fminf(v[2], v[3]));
  if (__ballot(least < 0x1p-96f)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) root[e] = root_of(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) root[e] = fast_sqrt(v[e]);
  }
}

// (The denominator is no subnormal number: the root of the smallest v above zero is 3.7e-23, and eps is none.)
__device__ __forceinline__ float next_param(const AdamwLaunch& launch, float p, float m, float root) {
  return p * launch.decay - launch.step_size * (m * fast_reciprocal(root * launch.root_scale + launch.eps));
}

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < INFINITY; }

// A parameter as it is stored: in bf16 by its random bits, if there are any.
template <class P>
__device__ __forceinline__ P stored_param(float p, bool stochastic, uint32_t word) {
  if constexpr (sizeof(P) == 2) {
    if (stochastic && is_finite(p)) return from_float<P>(__uint_as_float((__float_as_uint(p) + (mix(word ^ 0x5BF03635u) & 0xFFFFu)) & 0xFFFF0000u));
  }
  return from_float<P>(p);
}

__device__ __forceinline__ uint32_t word_of(uint64_t i, uint32_t key) { return mix((uint32_t)i + (uint32_t)(i >> 32) * 0x632BE5ABu + key); }

// ---- states in 8 bits -----------------------------------------------------------------------------
// The biased exponent of a block's scale from its largest value: the smallest power of two that keeps it
// within 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t scale_of(uint32_t largest_bits) {
  const int k = (int)((largest_bits + 0x1FFFFFu) >> 23) - 8;
  return k < 10 ? 10u : (uint32_t)k;
}

// The largest magnitude of a block, as bits, from the four values of each of its 8 lanes. As whole numbers the bits
// are ordered as the magnitudes are, with what is not finite on top: that counts for nothing here, and `odd` says
// whether any lane of the wavefront has it.
__device__ __forceinline__ uint32_t largest_of(const float (&x)[4], bool& odd) {
  const auto over_lanes = [](uint32_t top) {
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, top, 0xB1, 0xf, 0xf, true));
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, top, 0x4E, 0xf, 0xf, true));
    return max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, top, 0x141, 0xf, 0xf, true));
  };
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(fabsf(x[e])));
  const uint32_t all = over_lanes(top);
  odd = __ballot(all >= 0x7F800000u) != 0;
  if (!odd) return all;
  top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) top = max(top, is_finite(x[e]) ? __float_as_uint(fabsf(x[e])) : 0u);
  return over_lanes(top);
}

// The e4m3 value, as a float, beside |x| / 2^(scale - 127) that the 16 bits of `half` choose: the upper one where
// (half + 0.5) / 65536 is less than the share of the way. Below 2^-6 the codes lie 2^-9 apart, as they do in the
// binade above: 2^-6 is added there and taken away again.
//
// Where the expectation of the value is kept, the choice is an addition: 20 bits of the mantissa lie below a code's
// three, and they reach the code above where they and what is added make 2^20.
__device__ __forceinline__ float chosen_value(float x, float inverse_scale, uint32_t half) {
  const float size = fabsf(x) * inverse_scale;
  const float shift = size < 0x1p-6f ? 0x1p-6f : 0.0f;
  const uint32_t bits = __float_as_uint(size + shift) + (0x100000u - 9) - half * 16;
  return __uint_as_float(bits & 0xFFF00000u) - shift;
}

// Where that of the square v = x^2 is kept: with the codes a and a + s beside x the share is (v - a^2) / (s (2 a + s)), made
// from v itself: the root has been rounded, a's square is exact. What is not zero does not become zero. `eight` is 8 s,
// the power of two that x begins with.
__device__ __forceinline__ float chosen_root(float x, float v, float inverse_scale, uint32_t half) {
  float size = x * inverse_scale;
  size = size > 0 ? fmaxf(size, 0x1p-9f) : size;
  const float shift = size < 0x1p-6f ? 0x1p-6f : 0.0f;
  const uint32_t bits = __float_as_uint(size + shift);
  const float below = __uint_as_float(bits & 0xFFF00000u) - shift, eight = __uint_as_float(bits & 0x7F800000u);
  const float whole = ((float)half * 0x1p-22f + 0x1p-23f) * eight * (16 * below + eight);  // (half + 0.5) / 65536 of s (2 a + s)
  return whole < v * inverse_scale * inverse_scale - below * below ? below + 0.125f * eight : below;
}

// 2^(scale - 127). As an exponent 0 means zero and 255 infinity; with the highest bit of a mantissa they are 2^-127 and not a
// number, as E8M0 has them.
__device__ __forceinline__ float scale_value(uint32_t scale) { return __uint_as_float(scale << 23 | ((scale + 1) & 0xFE ? 0 : 0x400000)); }

// Four codes as values, times `factor`.
__device__ __forceinline__ void values_of(uint32_t codes, float factor, float (&x)[4]) {
  x[0] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 0) * factor;
  x[1] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 1) * factor;
  x[2] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 2) * factor;
  x[3] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 3) * factor;
}

// The codes of four values and the scale of their block. kRoots: the roots of `squares`, by the high halves of the words;
// else any values, by the low ones.
template <bool kRoots>
__device__ __forceinline__ uint32_t codes_of(const float (&x)[4], const float (&squares)[4], const uint32_t (&word)[4], uint32_t& scale) {
  bool odd;
  scale = scale_of(largest_of(x, odd));
  const float inverse = __uint_as_float((254u - scale) << 23);
  float c[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    c[e] = kRoots ? chosen_root(x[e], squares[e], inverse, word[e] >> 16) : copysignf(chosen_value(x[e], inverse, word[e] & 0xFFFFu), x[e]);
  const int low = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
  uint32_t codes = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], low, true);
  if (odd) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!is_finite(x[e])) codes = (codes & ~(0xFFu << 8 * e)) | 0x7Fu << 8 * e;  // not a number
  }
  return codes;
}

// ---- the step -------------------------------------------------------------------------------------
// kVectors times four elements to a lane, all of their loads before the first store; `elems` from element `first` on.
// C: the type of copies, or void where there are none.
template <class P, class G, class C, bool kEight, bool kStream, bool kWhole>
__device__ __forceinline__ void adamw_tile(const AdamwLaunch& launch, uint32_t k, uint64_t first, uint32_t elems) {
  constexpr AdamwShape kShape = adamw_shape(kEight);
  constexpr uint32_t kThreads = kShape.threads, kVectors = kShape.vectors;
  const float factor = factor_of(launch);
  const bool stochastic = sizeof(P) == 2 && launch.stochastic;
  const uint32_t key = kEight || stochastic ? mix(launch.seed + (launch.first_item + k) * 0x9E3779B1u) : 0;
  constexpr bool kCopies = !std::is_void_v<C>;
  typedef std::conditional_t<kCopies, C, bf16> Copy;
  const uint64_t* const words = launch.words + k * AdamwLaunch::words_of(kEight, kCopies) + 1;  // (AdamwLaunch::set)
  P* const param = reinterpret_cast<P*>(words[0]) + first;
  const G* const grad = reinterpret_cast<const G*>(words[1]) + first;
  typedef std::conditional_t<kEight, uint8_t, float> S;
  S* const m_state = reinterpret_cast<S*>(words[2]) + first;
  S* const v_state = reinterpret_cast<S*>(words[3]) + first;
  uint8_t* const m_scale = kEight ? reinterpret_cast<uint8_t*>(words[4]) + first / kBlock : nullptr;
  uint8_t* const v_scale = kEight ? reinterpret_cast<uint8_t*>(words[5]) + first / kBlock : nullptr;
  Copy* const copy = kCopies ? reinterpret_cast<Copy*>(words[kEight ? 6 : 4]) + first : nullptr;
  Four<P> p[kVectors];
  Four<G> g[kVectors];
  Four<S> m[kVectors], v[kVectors];
  uint32_t m_exponent[kVectors], v_exponent[kVectors];
#pragma unroll
  for (uint32_t u = 0; u < kVectors; ++u) {
    const uint32_t i = (u * kThreads + threadIdx.x) * 4, n = kWhole || i + 4 <= elems ? 4 : i < elems ? elems - i : 0;
    g[u].template load<kStream>(grad + i, n);
    p[u].template load<kStream>(param + i, n);
    m[u].template load<kStream>(m_state + i, n);
    v[u].template load<kStream>(v_state + i, n);
    if constexpr (kEight) {
      m_exponent[u] = n ? m_scale[i / kBlock] : 0;
      v_exponent[u] = n ? v_scale[i / kBlock] : 0;
    }
  }
#pragma unroll
  for (uint32_t u = 0; u < kVectors; ++u) {
    const uint32_t i = (u * kThreads + threadIdx.x) * 4, n = kWhole || i + 4 <= elems ? 4 : i < elems ? elems - i : 0;
    float m_now[4], v_now[4], root[4];
    uint32_t word[4];
    if constexpr (kEight) {
      values_of(__builtin_bit_cast(uint32_t, m[u].v), scale_value(m_exponent[u]) * launch.beta1, m_now);
      values_of(__builtin_bit_cast(uint32_t, v[u].v), scale_value(v_exponent[u]), root);
    }
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      const float gradient = to_float(g[u].v[e]) * factor;
      const float beta_m = kEight ? m_now[e] : (float)m[u].v[e] * launch.beta1, v_old = kEight ? root[e] * root[e] : (float)v[u].v[e];
      m_now[e] = beta_m + gradient * launch.one_minus_beta1;
      v_now[e] = v_old * launch.beta2 + gradient * gradient * launch.one_minus_beta2;
      if (kEight || stochastic) word[e] = word_of(first + i + e, key);
    }
    roots_of(v_now, root);
    Four<Copy> c;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      float q = next_param(launch, to_float(p[u].v[e]), m_now[e], root[e]);
      // The copy is the parameter's rounding: the compiler would make it of the unrounded difference, by an instruction
      // that subtracts into fp16.
      if constexpr (kCopies) asm("" : "+v"(q));
      p[u].v[e] = stored_param<P>(q, stochastic, word[e]);
      c.v[e] = from_float<Copy>(q);
      if constexpr (!kEight) {
        m[u].v[e] = m_now[e];
        v[u].v[e] = v_now[e];
      }
    }
    if constexpr (kEight) {  // (lanes without elements hold zeros, and come along to their block's largest value)
      m[u].v = __builtin_bit_cast(typename Four<S>::type, codes_of<false>(m_now, v_now, word, m_exponent[u]));
      v[u].v = __builtin_bit_cast(typename Four<S>::type, codes_of<true>(root, v_now, word, v_exponent[u]));
      if (n && threadIdx.x % (kBlock / 4) == 0) {
        m_scale[i / kBlock] = (uint8_t)m_exponent[u];
        v_scale[i / kBlock] = (uint8_t)v_exponent[u];
      }
    }
    p[u].template store<kStream>(param + i, n);
    m[u].template store<kStream>(m_state + i, n);
    v[u].template store<kStream>(v_state + i, n);
    if constexpr (kCopies) c.template store<false>(copy + i, n);
  }
}

template <class P, class G, class C, bool kEight, bool kStream>
__global__ __launch_bounds__(adamw_shape(kEight).threads) __attribute__((amdgpu_waves_per_eu(1, adamw_shape(kEight).waves))) void adamw_kernel(
    AdamwLaunch launch) {
  constexpr uint32_t kTile = adamw_shape(kEight).tile();
  const uint32_t k = item_of(launch, blockIdx.x);
  const uint64_t first = (uint64_t)(blockIdx.x - launch.first_tile[k]) * kTile, left = launch.words[k * AdamwLaunch::words_of(kEight, !std::is_void_v<C>)] - first;
  if (left >= kTile) adamw_tile<P, G, C, kEight, kStream, true>(launch, k, first, kTile);
  else adamw_tile<P, G, C, kEight, kStream, false>(launch, k, first, (uint32_t)left);
}

// As many values to a lane as 16 bytes hold: what is written is most of the work. (27.3 M values into bf16: 15.3 us, 5.4 TB/s;
// four values to a lane, whose stores are 8 bytes: 22.9.)
template <class T>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t* codes, const uint8_t* scales, T* values, uint64_t elems) {
  constexpr uint32_t kElems = Vector<T>::kElems;
  const uint64_t first = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * kElems;
  if (first + kElems <= elems) {
    typedef uint32_t Codes __attribute__((ext_vector_type(kElems / 4)));
    typedef Codes CodesAnywhere __attribute__((aligned(1)));
    const Codes c = *reinterpret_cast<const CodesAnywhere*>(codes + first);
    const float scale = scale_value(scales[first / kBlock]);
    typename Vector<T>::type out;
#pragma unroll
    for (uint32_t f = 0; f < kElems / 4; ++f) {
      float x[4];
      values_of(c[f], scale, x);
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) out[4 * f + e] = from_float<T>(x[e]);
    }
    *reinterpret_cast<typename Vector<T>::unaligned*>(values + first) = out;
  } else {
    for (uint64_t i = first; i < elems; ++i)
      values[i] = from_float<T>(__builtin_amdgcn_cvt_f32_fp8((int)codes[i], 0) * scale_value(scales[i / kBlock]));
  }
}

template <class Body>
int with_type(int32_t dtype, Body body) {
  return dtype == ODC_OPS_F32 ? body(float()) : dtype == ODC_OPS_BF16 ? body(bf16()) : body(f16());
}

}  // namespace

int launch_squared_norm(int32_t dtype, bool stream_past_caches, const SquaredNormLaunch& l, uint32_t blocks, double* partials, void* stream) {
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return launch(stream_past_caches ? squared_norm_kernel<T, true> : squared_norm_kernel<T, false>, blocks, 256, stream, l, partials);
  });
}

int launch_squared_norm_total(const double* partials, uint32_t n, float* result, void* stream) {
  return launch(squared_norm_total_kernel, 1, 256, stream, partials, n, result);
}

int launch_adamw(int32_t param, int32_t grad, int32_t copy, int32_t state_bits, bool stream_past_caches, const AdamwLaunch& l, void* stream) {
  return with_type(grad, [&](auto g) {
    const auto with_param = [&](auto p, auto c) {
      using P = decltype(p);
      using G = decltype(g);
      using C = std::remove_pointer_t<decltype(c)>;
      const auto kernel = state_bits == 8 ? (stream_past_caches ? adamw_kernel<P, G, C, true, true> : adamw_kernel<P, G, C, true, false>)
                                          : (stream_past_caches ? adamw_kernel<P, G, C, false, true> : adamw_kernel<P, G, C, false, false>);
      return launch(kernel, l.n_tiles, adamw_shape(state_bits == 8).threads, stream, l);
    };
    if (param == ODC_OPS_BF16) return with_param(bf16(), (void*)nullptr);
    if (copy == ODC_OPS_NONE) return with_param(float(), (void*)nullptr);
    return copy == ODC_OPS_F16 ? with_param(float(), (f16*)nullptr) : with_param(float(), (bf16*)nullptr);
  });
}

int launch_dequantize(const void* codes, const void* scales, void* values, uint64_t elems, int32_t dtype, void* stream) {
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr uint32_t kTile = 256 * Vector<T>::kElems;
    return launch(dequantize_kernel<T>, (uint32_t)((elems + kTile - 1) / kTile), 256, stream, static_cast<const uint8_t*>(codes),
                  static_cast<const uint8_t*>(scales), static_cast<T*>(values), elems);
  });
}

}  // namespace odc_ops_device
