/*
 * odc_ops.h — C ABI of libodc_ops.so, the operators of a training step around the ODC primitives on
 * MI355X (gfx950): layer norm forward and backward, the AdamW step over many tensors (states in fp32 or
 * in 8 bits) and the squared norm of many tensors.
 *
 * Conventions
 *   - Every function returns ODC_OPS_OK (0) or a negative odc_ops_status; nothing aborts the process.
 *     odc_ops_last_error() returns a thread-local, human-readable message for the last failure.
 *   - All launches are asynchronous on the hipStream_t passed as `stream` (NULL = the null stream), on
 *     the device that is current; nothing is allocated, copied or synchronised, so every call can be
 *     captured into a HIP graph.
 *   - Pointers are device pointers, aligned to the size of their element; no other alignment is asked
 *     for. Strides and sizes are in elements unless the name says `bytes`.
 *   - The sums of a call are made in an order that depends on the sizes alone: the same inputs give the
 *     same bits.
 */
#ifndef ODC_OPS_H_
#define ODC_OPS_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ODC_OPS_ABI_VERSION 2

typedef enum odc_ops_status {
  ODC_OPS_OK = 0,
  ODC_OPS_ERR_INVALID = -1,    /* bad argument (null, misaligned, too large, workspace too small, ...) */
  ODC_OPS_ERR_HIP = -3,        /* a HIP runtime call failed (message carries hipGetErrorString) */
  ODC_OPS_ERR_UNSUPPORTED = -4 /* dtype combination not implemented */
} odc_ops_status;

/* The values of odc_dtype in odc_hip.h. */
typedef enum odc_ops_dtype {
  ODC_OPS_NONE = -1,
  ODC_OPS_BF16 = 0,
  ODC_OPS_F16 = 1,
  ODC_OPS_F32 = 2
} odc_ops_dtype;

/* -- layer norm -------------------------------------------------------------------------------------
 * Rows of `width` elements (2^26 at most); a row's elements are neighbours, rows lie `..._stride` elements apart
 * (any stride, 0 included, for what is read). What is written is dense: row i at i * width.
 *
 *   total  = input + residual, rounded to `dtype`     (only with a residual; else total = input)
 *   output = (total - mean) * rstd * weight + bias,   rstd = 1 / sqrt(variance + eps)
 *
 * mean and rstd (fp32, one per row) may be NULL; weight and bias (of `weight_dtype`, which is `dtype`
 * or fp32) too: without weight 1 is meant, without bias 0. */
typedef struct odc_norm_forward {
  const void* input;
  const void* residual; /* NULL: none */
  const void* weight;
  const void* bias;
  void* output;
  void* total; /* written exactly when there is a residual */
  float* mean;
  float* rstd;
  uint64_t rows, width;
  uint64_t input_stride, residual_stride;
  int32_t dtype, weight_dtype;
  float eps;
} odc_norm_forward;

int odc_layer_norm(const odc_norm_forward* call, void* stream);

/* `normalised` is what forward normalised: its input, or its total. With h = grad_output * weight and
 * z = (normalised - mean) * rstd:
 *
 *   grad_input  = rstd * (h - mean(h) - z * mean(h * z)) (+ grad_total)
 *   grad_weight = sum over rows of grad_output * z,   grad_bias = sum over rows of grad_output
 *
 * Any of the three may be NULL and is not computed. With a residual, grad_total is the gradient of the
 * handed on total (NULL: zero) and grad_input is the gradient of both the input and the residual.
 * `workspace` takes odc_layer_norm_backward_workspace() bytes, aligned to 16. */
typedef struct odc_norm_backward {
  const void* grad_output;
  const void* grad_total; /* NULL: none */
  const void* normalised;
  const void* weight; /* NULL: 1 */
  const float* mean;
  const float* rstd;
  void* grad_input;
  void* grad_weight;
  void* grad_bias;
  void* workspace;
  uint64_t workspace_bytes;
  uint64_t rows, width;
  uint64_t grad_output_stride, grad_total_stride, normalised_stride;
  int32_t dtype, weight_dtype;
} odc_norm_backward;

uint64_t odc_layer_norm_backward_workspace(uint64_t rows, uint64_t width, int32_t dtype);
int odc_layer_norm_backward(const odc_norm_backward* call, void* stream);

/* -- squared norm -----------------------------------------------------------------------------------
 * *result (fp32) = the sum of the squares of all elements of all tensors. `workspace` takes
 * odc_squared_norm_workspace() bytes, aligned to 8. */
typedef struct odc_span_item {
  const void* data;
  uint64_t elems;
} odc_span_item;

uint64_t odc_squared_norm_workspace(const odc_span_item* items, uint32_t n_items, int32_t dtype);
int odc_squared_norm(const odc_span_item* items, uint32_t n_items, int32_t dtype, void* workspace,
                     uint64_t workspace_bytes, float* result, void* stream);

/* -- AdamW ------------------------------------------------------------------------------------------
 * For every element of every tensor, in fp32, with t = step:
 *
 *   g = grad * grad_scale * c,   c = min(1, max_norm / (grad_scale * sqrt(*squared_norm) + 1e-6))
 *   m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
 *   p = p (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 *
 * (eps is 0 or a normal fp32 number; c = 1 where squared_norm is NULL). `copy`, where it is given, receives p in copy_dtype.
 *
 * state_bits 32: exp_avg and exp_avg_sq are fp32, m and v.
 * state_bits 8: exp_avg and exp_avg_sq hold m and the ROOT of v as OCP e4m3 values; 32 neighbouring
 * elements share a power of two, whose exponent plus 127 is a byte of exp_avg_scale / exp_avg_sq_scale
 * ((elems + 31) / 32 bytes each). A scale is the smallest power of two, not below 2^-117, that keeps the
 * block's largest value within 448; what is not finite is stored as NaN and counts for no scale.
 * A value x between two codes is stored as one of them by a random number of 16 bits, so that the
 * expectation is m, and that of the root's square v (an average that moves by less than half a code in
 * a step would otherwise never move); a v > 0 is stored as the smallest code at least (the next step
 * would divide by eps alone). All zeros, scales included, is the state to begin with.
 *
 * The random numbers are the caller's by `seed`: element i of tensor k of the call has
 *   word = mix(lo32(i) + hi32(i) * 0x632BE5AB + mix(lo32(seed) + k * 0x9E3779B1)),
 * the low half for m, the high half for the root; mix(x): x ^= x >> 16, x *= 0xB7E15163, x ^= x >> 15,
 * x *= 0x9E3779B1, x ^= x >> 16, in 32 bits. A half h takes the upper code where (h + 0.5) / 65536 is less
 * than the share of the way between the two (their squares, for the root). With `stochastic` set, parameters in bf16 are rounded by
 * the low half of mix(word ^ 0x5BF03635) as well, added below the bits that stay; without it, and
 * copies always, to the nearest even value.
 *
 * Types: parameters fp32 or bf16; gradients fp32, bf16 or fp16; copies bf16 or fp16, of fp32 parameters
 * only. The tensors of one call do not overlap. */
typedef struct odc_adamw_item {
  void* param;
  const void* grad;
  void* exp_avg;
  void* exp_avg_sq;
  void* exp_avg_scale;    /* 8 bits only */
  void* exp_avg_sq_scale; /* 8 bits only */
  void* copy;             /* NULL: none */
  uint64_t elems;
} odc_adamw_item;

typedef struct odc_adamw_numbers {
  double lr, beta1, beta2, eps, weight_decay, grad_scale, max_norm;
  const float* squared_norm; /* on the device; NULL: no clipping */
  uint64_t step;             /* 1 for the first */
  uint32_t seed;
  int32_t stochastic;
  int32_t param_dtype, grad_dtype, copy_dtype, state_bits;
} odc_adamw_numbers;

int odc_adamw(const odc_adamw_item* items, uint32_t n_items, const odc_adamw_numbers* numbers, void* stream);
/* What odc_adamw would refuse, without a launch: for a step of several calls, all of which are to be made or none. */
int odc_adamw_check(const odc_adamw_item* items, uint32_t n_items, const odc_adamw_numbers* numbers);

/* values[i] = codes[i] * 2^(scales[i / 32] - 127), in `dtype`; a scale of 255 is not a number. */
int odc_dequantize_blocks(const void* codes, const void* scales, void* values, uint64_t elems, int32_t dtype,
                          void* stream);

const char* odc_ops_last_error(void);
int odc_ops_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif /* ODC_OPS_H_ */
