// odc_ops_host.cpp — the host side of libodc_ops.so: the C ABI of include/odc_ops.h, its checks and the launch
// plans. Plain C++: everything HIP is behind namespace odc_ops_device (odc_ops_launch.h).
#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <limits>

#include "odc_ops.h"
#include "odc_ops_launch.h"

namespace {

using namespace odc_ops_launch;

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int launched(int e) {
  return e == 0 ? ODC_OPS_OK : fail(ODC_OPS_ERR_HIP, "kernel launch failed: %s", odc_ops_device::error_string(e));
}

bool aligned(const void* p, uint64_t bytes) { return (uintptr_t)p % bytes == 0; }

uint64_t ceil_div(uint64_t a, uint64_t b) { return a / b + (a % b != 0); }

// The last byte of `rows` rows at `stride` must be addressable in 63 bits.
bool spans_too_much(uint64_t rows, uint64_t stride, uint64_t width) {
  constexpr uint64_t kMost = uint64_t(1) << 60;
  return width > kMost || rows > kMost || (rows && stride > kMost / rows);
}

constexpr uint64_t kLastLevelCache = uint64_t(256) << 20;

// ---- layer norm -----------------------------------------------------------------------------------
// The pass over groups has 256 threads for 32 of twice as many columns, and a dispatch counts them in 32 bits.
constexpr uint64_t kMostColumns = uint64_t(1) << 26;
static_assert(2 * kMostColumns / kGroupColumns <= most_workgroups(256), "too many workgroups");

int check_norm(uint64_t rows, uint64_t width, int32_t dtype, int32_t weight_dtype) {
  if (!is_float_type(dtype) || !is_float_type(weight_dtype)) return fail(ODC_OPS_ERR_UNSUPPORTED, "unknown dtype %d or %d", dtype, weight_dtype);
  if (weight_dtype != dtype && weight_dtype != ODC_OPS_F32)
    return fail(ODC_OPS_ERR_UNSUPPORTED, "weights have the dtype of the input or fp32");
  if (width > kMostColumns) return fail(ODC_OPS_ERR_INVALID, "rows of %llu elements are too long", (unsigned long long)width);
  if (spans_too_much(rows, width, width)) return fail(ODC_OPS_ERR_INVALID, "sizes overflow: %llu rows of %llu", (unsigned long long)rows, (unsigned long long)width);
  return ODC_OPS_OK;
}

int check_rows(const char* name, const void* p, uint64_t rows, uint64_t width, uint64_t stride, int32_t dtype, bool needed = true) {
  if (!p) return needed ? fail(ODC_OPS_ERR_INVALID, "%s is NULL", name) : ODC_OPS_OK;
  if (!aligned(p, bytes_of(dtype))) return fail(ODC_OPS_ERR_INVALID, "%s is not aligned to its element", name);
  if (spans_too_much(rows, stride, width)) return fail(ODC_OPS_ERR_INVALID, "the stride of %s overflows", name);
  return ODC_OPS_OK;
}

#define ODC_OPS_TRY(expr)                          \
  do {                                             \
    const int rc_ = (expr);                        \
    if (rc_ != ODC_OPS_OK) return rc_;             \
  } while (0)

constexpr uint64_t kCus = 256;

// Whether rows of whole 16 byte vectors start at multiples of 16 bytes.
bool rows_of_vectors(const void* p, uint64_t stride, int32_t dtype) { return aligned(p, 16) && stride * bytes_of(dtype) % 16 == 0; }

// What a pass reads and writes beyond the last-level cache's 256 MB is streamed past the caches: nothing of it would be
// found again. us, in the caches / streamed: 16384 x 14336 bf16 with a residual (1.9 GB a pass) forward 336 / 326,
// backward 380 / 330; 4096 x 4096 (134 MB) 24.7 / 30.0 and 31.8 / 33.7.
// (A wavefront has one row or a part of one: lanes is 64 at least.)
RowAccess access_of(bool vectors, const NormShape& shape, uint64_t rows, uint64_t width, int32_t dtype, int tensors) {
  if (!vectors || shape.lanes < 64) return kPlainRows;
  return rows * width * bytes_of(dtype) > kLastLevelCache / tensors ? kStreamRows : kBufferRows;
}

RowAccess access_of(const odc_norm_forward& c, const NormShape& shape) {
  const bool vectors = rows_of_vectors(c.input, c.input_stride, c.dtype) && rows_of_vectors(c.residual, c.residual_stride, c.dtype) &&
                       rows_of_vectors(c.output, c.width, c.dtype) && rows_of_vectors(c.total, c.width, c.dtype) && aligned(c.weight, 16) &&
                       aligned(c.bias, 16);
  return access_of(vectors, shape, c.rows, c.width, c.dtype, c.residual ? 4 : 2);
}

RowAccess access_of(const odc_norm_backward& c, const NormShape& shape) {
  const bool vectors = rows_of_vectors(c.grad_output, c.grad_output_stride, c.dtype) && rows_of_vectors(c.grad_total, c.grad_total_stride, c.dtype) &&
                       rows_of_vectors(c.normalised, c.normalised_stride, c.dtype) && rows_of_vectors(c.grad_input, c.width, c.dtype) &&
                       aligned(c.weight, 16);
  return access_of(vectors, shape, c.rows, c.width, c.dtype, 2 + (c.grad_total != nullptr) + (c.grad_input != nullptr));
}

NormForwardPlan forward_plan(uint64_t rows, uint64_t width, int32_t dtype) {
  NormForwardPlan plan = {};
  plan.shape = shape_of(kForwardShapes, width, dtype);
  uint64_t rows_at_once = 1, most = 8 * kCus;
  if (plan.shape.lanes) {
    const uint32_t threads = std::max(kForwardThreads, plan.shape.lanes);
    rows_at_once = threads / plan.shape.lanes;
    most = 2048 / threads * kCus;
  }
  plan.blocks = (uint32_t)std::min(ceil_div(rows, rows_at_once), most);
  return plan;
}

NormBackwardPlan backward_plan(uint64_t rows, uint64_t width, int32_t dtype) {
  NormBackwardPlan plan = {};
  plan.shape = dtype == ODC_OPS_F32 ? shape_of(kBackwardShapes32, width, dtype) : shape_of(kBackwardShapes16, width, dtype);
  plan.row_blocks = (uint32_t)std::min<uint64_t>(rows, 8 * kCus);
  if (plan.shape.lanes) {
    const uint64_t rounds = ceil_div(rows, kBackwardThreads / plan.shape.lanes);
    plan.groups = rows && rounds <= kRoundsAlone ? 1 : (uint32_t)std::min(rounds, kCus);
    plan.rows_per_group = 0;
  } else {
    // The pass over columns: a row at least for each wavefront of a group, and no more groups, whose sums go to memory and back,
    // than 1024 workgroups need, or 32 rows to a wavefront in long columns. us of the backward pass in bf16 by this rule /
    // with up to 256 groups / with 1024 workgroups whatever the rows: 1000 x 20000 49 / 61 / 49, 4096 x 20000 196 / 210 / 200,
    // 100000 x 20000 4417 / 4420 / 4977, 256 x 1000000 1042 / 1066 / 1027. (A group for every row, of which a wavefront in
    // four has any, makes a workspace of four times the input: 300 x 20000 39 instead of 25.)
    constexpr uint64_t kWaves = kWideThreads / 64, kWorkgroups = 1024, kRows = 32;
    const uint64_t tiles = ceil_div(width, 64 * (16 / bytes_of(dtype)));
    const uint64_t groups = std::min({ceil_div(rows, kWaves), std::max(ceil_div(kWorkgroups, tiles), ceil_div(rows, kWaves * kRows)), kCus});
    plan.rows_per_group = rows ? ceil_div(rows, groups) : 1;
    plan.groups = (uint32_t)ceil_div(rows, plan.rows_per_group);
  }
  return plan;
}

// ---- lists ----------------------------------------------------------------------------------------
// Fills a launch's table with items from `at` on; returns the first item that is not in it.
template <class Launch, class Item>
uint32_t fill_table(Launch& launch, const Item* items, uint32_t n_items, uint32_t at, uint32_t most_items, uint32_t tile, uint32_t threads) {
  launch.n_items = launch.n_tiles = 0;
  while (at < n_items && launch.n_items < most_items) {
    const uint64_t tiles = ceil_div(items[at].elems, tile);
    if (tiles > most_workgroups(threads) - launch.n_tiles) break;  // (one tensor alone always fits: check_elems)
    launch.first_tile[launch.n_items] = launch.n_tiles;
    launch.set(launch.n_items++, items[at++]);
    launch.n_tiles += (uint32_t)tiles;
  }
  launch.first_tile[launch.n_items] = launch.n_tiles;
  return at;
}

int check_elems(uint64_t elems, uint32_t i, uint32_t tile, uint32_t threads) {
  if (ceil_div(elems, tile) > most_workgroups(threads)) return fail(ODC_OPS_ERR_INVALID, "item %u: %llu elements are too many", i, (unsigned long long)elems);
  return ODC_OPS_OK;
}

template <class Item>
uint64_t all_elems(const Item* items, uint32_t n_items) {
  uint64_t sum = 0;
  for (uint32_t i = 0; i < n_items; ++i) sum += items[i].elems;
  return sum;
}

uint32_t partials_of(uint32_t n_tiles) { return std::min(n_tiles, kMostPartials); }

}  // namespace

extern "C" {

const char* odc_ops_last_error(void) { return g_err; }
int odc_ops_abi_version(void) { return ODC_OPS_ABI_VERSION; }

int odc_layer_norm(const odc_norm_forward* call, void* stream) {
  if (!call) return fail(ODC_OPS_ERR_INVALID, "call is NULL");
  const odc_norm_forward& c = *call;
  ODC_OPS_TRY(check_norm(c.rows, c.width, c.dtype, c.weight_dtype));
  if (!c.rows || !c.width) return ODC_OPS_OK;
  ODC_OPS_TRY(check_rows("input", c.input, c.rows, c.width, c.input_stride, c.dtype));
  ODC_OPS_TRY(check_rows("residual", c.residual, c.rows, c.width, c.residual_stride, c.dtype, false));
  ODC_OPS_TRY(check_rows("output", c.output, c.rows, c.width, c.width, c.dtype));
  ODC_OPS_TRY(check_rows("total", c.total, c.rows, c.width, c.width, c.dtype, c.residual != nullptr));
  if (c.total && !c.residual) return fail(ODC_OPS_ERR_INVALID, "total without residual");
  ODC_OPS_TRY(check_rows("weight", c.weight, 1, c.width, c.width, c.weight_dtype, false));
  ODC_OPS_TRY(check_rows("bias", c.bias, 1, c.width, c.width, c.weight_dtype, false));
  if (!aligned(c.mean, 4) || !aligned(c.rstd, 4)) return fail(ODC_OPS_ERR_INVALID, "mean or rstd is not aligned to its element");
  NormForwardPlan plan = forward_plan(c.rows, c.width, c.dtype);
  plan.access = access_of(c, plan.shape);
  return launched(odc_ops_device::launch_norm_forward(c, plan, stream));
}

uint64_t odc_layer_norm_backward_workspace(uint64_t rows, uint64_t width, int32_t dtype) {
  if (check_norm(rows, width, dtype, ODC_OPS_F32) != ODC_OPS_OK || !rows || !width) return 0;
  const NormBackwardPlan plan = backward_plan(rows, width, dtype);
  return plan.one_launch() ? 0 : (uint64_t)plan.groups * 2 * width * sizeof(float);
}

int odc_layer_norm_backward(const odc_norm_backward* call, void* stream) {
  if (!call) return fail(ODC_OPS_ERR_INVALID, "call is NULL");
  const odc_norm_backward& c = *call;
  ODC_OPS_TRY(check_norm(c.rows, c.width, c.dtype, c.weight_dtype));
  if (!c.width || (!c.grad_input && !c.grad_weight && !c.grad_bias)) return ODC_OPS_OK;
  ODC_OPS_TRY(check_rows("grad_weight", c.grad_weight, 1, c.width, c.width, c.weight_dtype, false));
  ODC_OPS_TRY(check_rows("grad_bias", c.grad_bias, 1, c.width, c.width, c.weight_dtype, false));
  if (c.rows) {
    ODC_OPS_TRY(check_rows("grad_output", c.grad_output, c.rows, c.width, c.grad_output_stride, c.dtype));
    ODC_OPS_TRY(check_rows("grad_total", c.grad_total, c.rows, c.width, c.grad_total_stride, c.dtype, false));
    ODC_OPS_TRY(check_rows("normalised", c.normalised, c.rows, c.width, c.normalised_stride, c.dtype));
    ODC_OPS_TRY(check_rows("grad_input", c.grad_input, c.rows, c.width, c.width, c.dtype, false));
    ODC_OPS_TRY(check_rows("weight", c.weight, 1, c.width, c.width, c.weight_dtype, false));
    if (!c.mean || !c.rstd || !aligned(c.mean, 4) || !aligned(c.rstd, 4)) return fail(ODC_OPS_ERR_INVALID, "mean or rstd is NULL or not aligned");
  }
  if (c.grad_weight || c.grad_bias) {
    const uint64_t need = odc_layer_norm_backward_workspace(c.rows, c.width, c.dtype);
    if (need && (!c.workspace || c.workspace_bytes < need)) return fail(ODC_OPS_ERR_INVALID, "the workspace needs %llu bytes", (unsigned long long)need);
    if (!aligned(c.workspace, 16)) return fail(ODC_OPS_ERR_INVALID, "the workspace is not aligned to 16 bytes");
  }
  NormBackwardPlan plan = backward_plan(c.rows, c.width, c.dtype);
  plan.access = access_of(c, plan.shape);
  return launched(odc_ops_device::launch_norm_backward(c, plan, stream));
}

// A partial sum for every workgroup: as many as tiles, at most kMostPartials for each launch.
uint64_t odc_squared_norm_workspace(const odc_span_item* items, uint32_t n_items, int32_t dtype) {
  if (!items || !is_float_type(dtype)) return 0;
  uint64_t tiles = 0;
  for (uint32_t i = 0; i < n_items; ++i) {
    if (check_elems(items[i].elems, i, kNormTile, kNormThreads) != ODC_OPS_OK) return 0;
    tiles += ceil_div(items[i].elems, kNormTile);
  }
  const uint64_t launches = ceil_div(n_items, kNormItems) + 2 * (tiles / most_workgroups(kNormThreads));
  return std::min(tiles, launches * kMostPartials) * sizeof(double);
}

int odc_squared_norm(const odc_span_item* items, uint32_t n_items, int32_t dtype, void* workspace, uint64_t workspace_bytes, float* result,
                     void* stream) {
  if (!result || !aligned(result, 4)) return fail(ODC_OPS_ERR_INVALID, "result is NULL or not aligned");
  if (!items && n_items) return fail(ODC_OPS_ERR_INVALID, "items is NULL");
  if (!is_float_type(dtype)) return fail(ODC_OPS_ERR_UNSUPPORTED, "unknown dtype %d", dtype);
  for (uint32_t i = 0; i < n_items; ++i) {
    ODC_OPS_TRY(check_elems(items[i].elems, i, kNormTile, kNormThreads));
    if (!items[i].elems) continue;
    if (!items[i].data || !aligned(items[i].data, bytes_of(dtype))) return fail(ODC_OPS_ERR_INVALID, "item %u: data is NULL or not aligned to its element", i);
    if ((uint64_t)(uintptr_t)items[i].data >> 48) return fail(ODC_OPS_ERR_INVALID, "item %u: an address above 48 bits is no address of a GPU's", i);
  }
  const uint64_t need = n_items ? odc_squared_norm_workspace(items, n_items, dtype) : 0;
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 8)))
    return fail(ODC_OPS_ERR_INVALID, "the workspace needs %llu bytes, aligned to 8", (unsigned long long)need);
  if (need / sizeof(double) > 0xffffffffu) return fail(ODC_OPS_ERR_INVALID, "too many items");
  const bool past_caches = all_elems(items, n_items) > kLastLevelCache / bytes_of(dtype);
  double* partials = static_cast<double*>(workspace);
  uint32_t done = 0;
  SquaredNormLaunch launch;
  for (uint32_t at = 0; at < n_items;) {
    at = fill_table(launch, items, n_items, at, kNormItems, kNormTile, kNormThreads);
    const uint32_t blocks = partials_of(launch.n_tiles);
    if (!blocks) continue;
    ODC_OPS_TRY(launched(odc_ops_device::launch_squared_norm(dtype, past_caches, launch, blocks, partials + done, stream)));
    done += blocks;
  }
  return launched(odc_ops_device::launch_squared_norm_total(partials, done, result, stream));
}

int odc_adamw_check(const odc_adamw_item* items, uint32_t n_items, const odc_adamw_numbers* numbers) {
  if (!numbers) return fail(ODC_OPS_ERR_INVALID, "numbers is NULL");
  if (!items && n_items) return fail(ODC_OPS_ERR_INVALID, "items is NULL");
  const odc_adamw_numbers& a = *numbers;
  if (a.state_bits != 8 && a.state_bits != 32) return fail(ODC_OPS_ERR_UNSUPPORTED, "states have 32 bits or 8, not %d", a.state_bits);
  if ((a.param_dtype != ODC_OPS_F32 && a.param_dtype != ODC_OPS_BF16) || !is_float_type(a.grad_dtype))
    return fail(ODC_OPS_ERR_UNSUPPORTED, "parameters are fp32 or bf16, gradients fp32, bf16 or fp16");
  if (a.copy_dtype != ODC_OPS_NONE && (a.param_dtype != ODC_OPS_F32 || (a.copy_dtype != ODC_OPS_BF16 && a.copy_dtype != ODC_OPS_F16)))
    return fail(ODC_OPS_ERR_UNSUPPORTED, "copies are bf16 or fp16, of fp32 parameters");
  if (a.step < 1) return fail(ODC_OPS_ERR_INVALID, "the first step is 1");
  if (!(a.beta1 >= 0 && a.beta1 < 1 && a.beta2 >= 0 && a.beta2 < 1)) return fail(ODC_OPS_ERR_INVALID, "the betas lie in [0, 1)");
  if (!(a.eps >= 0) || !(a.lr >= 0) || !(a.weight_decay >= 0) || !std::isfinite(a.eps) || !std::isfinite(a.lr) || !std::isfinite(a.weight_decay))
    return fail(ODC_OPS_ERR_INVALID, "lr, eps and weight_decay are finite and not negative");
  // (The kernel's reciprocal takes a subnormal number for zero: 0 / eps would not be a number.)
  if (a.eps > 0 && (float)a.eps < std::numeric_limits<float>::min())
    return fail(ODC_OPS_ERR_INVALID, "eps is 0 or at least 1.18e-38, the smallest normal fp32 number");
  if (!(a.grad_scale >= 0) || !std::isfinite(a.grad_scale)) return fail(ODC_OPS_ERR_INVALID, "grad_scale is finite and not negative");
  if (a.squared_norm && (!(a.max_norm >= 0) || !aligned(a.squared_norm, 4)))
    return fail(ODC_OPS_ERR_INVALID, "max_norm is not negative, squared_norm aligned to its element");
  const AdamwShape shape = adamw_shape(a.state_bits == 8);
  for (uint32_t i = 0; i < n_items; ++i) {
    const odc_adamw_item& it = items[i];
    if (!it.elems) continue;
    ODC_OPS_TRY(check_elems(it.elems, i, shape.tile(), shape.threads));
    if (!it.param || !it.grad || !it.exp_avg || !it.exp_avg_sq) return fail(ODC_OPS_ERR_INVALID, "item %u: a pointer is NULL", i);
    if (a.state_bits == 8 && (!it.exp_avg_scale || !it.exp_avg_sq_scale)) return fail(ODC_OPS_ERR_INVALID, "item %u: scales are NULL", i);
    if ((a.copy_dtype != ODC_OPS_NONE) != (it.copy != nullptr)) return fail(ODC_OPS_ERR_INVALID, "item %u: copies of all tensors or of none", i);
    if (!aligned(it.param, bytes_of(a.param_dtype)) || !aligned(it.grad, bytes_of(a.grad_dtype)) || !aligned(it.copy, 2) ||
        (a.state_bits == 32 && (!aligned(it.exp_avg, 4) || !aligned(it.exp_avg_sq, 4))))
      return fail(ODC_OPS_ERR_INVALID, "item %u: a pointer is not aligned to its element", i);
  }
  return ODC_OPS_OK;
}

int odc_adamw(const odc_adamw_item* items, uint32_t n_items, const odc_adamw_numbers* numbers, void* stream) {
  ODC_OPS_TRY(odc_adamw_check(items, n_items, numbers));
  const odc_adamw_numbers& a = *numbers;
  const AdamwShape shape = adamw_shape(a.state_bits == 8);
  const uint32_t bytes = 2 * bytes_of(a.param_dtype) + bytes_of(a.grad_dtype) + (a.state_bits == 32 ? 16 : 4);
  const bool past_caches = all_elems(items, n_items) > kLastLevelCache / bytes;
  const double t = (double)a.step;
  AdamwLaunch launch;
  launch.beta1 = (float)a.beta1;
  launch.beta2 = (float)a.beta2;
  launch.one_minus_beta1 = (float)(1 - a.beta1);
  launch.one_minus_beta2 = (float)(1 - a.beta2);
  launch.decay = (float)(1 - a.lr * a.weight_decay);
  launch.step_size = (float)(a.lr / (1 - std::pow(a.beta1, t)));
  launch.root_scale = (float)(1 / std::sqrt(1 - std::pow(a.beta2, t)));
  launch.eps = (float)a.eps;
  launch.grad_scale = (float)a.grad_scale;
  launch.max_norm = (float)a.max_norm;
  launch.squared_norm = a.squared_norm;
  launch.seed = a.seed;
  launch.stochastic = a.stochastic != 0;
  launch.words_per_item = AdamwLaunch::words_of(a.state_bits == 8, a.copy_dtype != ODC_OPS_NONE);
  for (uint32_t at = 0; at < n_items;) {
    launch.first_item = at;
    at = fill_table(launch, items, n_items, at, kAdamwWords / launch.words_per_item, shape.tile(), shape.threads);
    if (!launch.n_tiles) continue;
    ODC_OPS_TRY(launched(odc_ops_device::launch_adamw(a.param_dtype, a.grad_dtype, a.copy_dtype, a.state_bits, past_caches, launch, stream)));
  }
  return ODC_OPS_OK;
}

int odc_dequantize_blocks(const void* codes, const void* scales, void* values, uint64_t elems, int32_t dtype, void* stream) {
  if (!is_float_type(dtype)) return fail(ODC_OPS_ERR_UNSUPPORTED, "unknown dtype %d", dtype);
  if (!elems) return ODC_OPS_OK;
  if (!codes || !scales || !values || !aligned(values, bytes_of(dtype))) return fail(ODC_OPS_ERR_INVALID, "a pointer is NULL or not aligned");
  if (ceil_div(elems, 1024) > most_workgroups(256)) return fail(ODC_OPS_ERR_INVALID, "%llu elements are too many", (unsigned long long)elems);
  return launched(odc_ops_device::launch_dequantize(codes, scales, values, elems, dtype, stream));
}

}  // extern "C"
