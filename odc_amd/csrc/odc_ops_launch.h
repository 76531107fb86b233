// odc_ops_launch.h — what the host side of libodc_ops.so (odc_ops_host.cpp, plain C++: the C ABI, the checks
// and the launch plans) hands to its device side (odc_norm_kernels.hip, odc_adamw_kernels.hip). The
// descriptors travel BY VALUE in the kernel-argument segment. A second implementation of namespace
// odc_ops_device without a device (tests/cpu/no_ops_device.cpp) lets the host side run under
// AddressSanitizer and UBSan on the CPU.
#ifndef ODC_OPS_LAUNCH_H_
#define ODC_OPS_LAUNCH_H_

#include <stddef.h>
#include <stdint.h>

#include "odc_ops.h"

namespace odc_ops_launch {

inline bool is_float_type(int32_t dtype) { return dtype == ODC_OPS_BF16 || dtype == ODC_OPS_F16 || dtype == ODC_OPS_F32; }
inline uint32_t bytes_of(int32_t dtype) { return dtype == ODC_OPS_F32 ? 4 : 2; }

// ---- layer norm -----------------------------------------------------------------------------------
// A row is held in the registers of `lanes` lanes, `vectors` vectors of 16 bytes each; rows wider than the last shape
// are passed over three times. The backward pass has sums for weight and bias beside them, 16 or 8 registers to a vector.
struct NormShape {
  uint32_t lanes, vectors;
};
constexpr NormShape kForwardShapes[] = {{16, 1}, {32, 1}, {64, 1}, {64, 2}, {256, 1}, {256, 2}, {512, 2}, {1024, 2}, {1024, 4}};
constexpr NormShape kBackwardShapes16[] = {{16, 1}, {32, 1}, {64, 1}, {128, 1}, {256, 1}, {512, 1}, {1024, 1}, {1024, 2}};
constexpr NormShape kBackwardShapes32[] = {{16, 1}, {32, 1}, {64, 1}, {128, 1}, {256, 1}, {512, 1}, {1024, 1}, {1024, 2}, {1024, 4}};
constexpr uint32_t kForwardThreads = 256;  // of a workgroup; where a row takes more lanes, as many as those
// One workgroup to a CU: each writes its sums of all columns, and a second launch reads them. (Two of 512 threads: level
// for long passes, 33.8 instead of 32.0 us for 4096 x 4096.)
constexpr uint32_t kBackwardThreads = 1024;
constexpr uint32_t kWideThreads = 256;  // of one for wide rows
// Rows ahead of the one that a backward pass works on, with one vector to a lane. us for 16384 x 4096 bf16 with 1, 2, 3:
// 86.5, 74.2, 75.9; 65536 x 1024: 82.6, 69.8, 70.7.
constexpr int kRowsAhead = 2;

// The first of `shapes` that holds a row; lanes 0: none does, or the row is less than a vector.
template <size_t n>
inline NormShape shape_of(const NormShape (&shapes)[n], uint64_t width, int32_t dtype) {
  if (width < 16 / bytes_of(dtype)) return {0, 0};
  for (const NormShape& s : shapes)
    if (width <= (uint64_t)s.lanes * s.vectors * (16 / bytes_of(dtype))) return s;
  return {0, 0};
}

// How rows in registers are read and written (Piece in odc_norm_kernels.hip, access_of in odc_ops_host.cpp).
enum RowAccess : uint32_t { kPlainRows, kBufferRows, kStreamRows };

struct NormForwardPlan {
  NormShape shape;
  RowAccess access;
  uint32_t blocks;
};

// The gradients of weight and bias are sums over the rows. `groups` workgroups add up rows of their own, each
// into its row of the workspace ([groups][2][width] floats), and a second launch adds the groups.
struct NormBackwardPlan {
  NormShape shape;
  RowAccess access;
  uint32_t groups;
  uint32_t row_blocks;      // wide rows: workgroups of the pass over rows
  uint64_t rows_per_group;  // wide rows: of the pass over columns

  // One workgroup alone has nothing to add.
  bool one_launch() const { return shape.lanes && groups == 1; }
};
// A few rows have one workgroup: up to four rounds of them take less than a launch and the workspace do.
constexpr uint32_t kRoundsAlone = 4;
constexpr uint32_t kGroupColumns = 32;  // columns of one workgroup of the pass over groups

// ---- lists of tensors -----------------------------------------------------------------------------
// A dispatch counts its work-items in 32 bits.
constexpr uint32_t most_workgroups(uint32_t threads) { return 0xffffffffu / threads; }

// A launch has a table of its tensors and the number of the first tile of each.
constexpr uint32_t kNormItems = 320;
constexpr uint32_t kNormThreads = 256;
constexpr uint32_t kNormTile = 8192;  // elements of a tile of the squared norm
constexpr uint32_t kMostPartials = 2048;
struct SquaredNormLaunch {
  uint32_t n_items, n_tiles;
  uint32_t first_tile[kNormItems + 1];
  // An item in 8 bytes, for a table of 320: its address (of 48 bits), and below it the elements of its last tile.
  uint64_t places[kNormItems];

  void set(uint32_t k, const odc_span_item& item) {
    const uint64_t last = item.elems ? (item.elems - 1) % kNormTile + 1 : 0;
    places[k] = (uint64_t)(uintptr_t)item.data << 16 | last;
  }
};
static_assert(sizeof(SquaredNormLaunch) <= 3900, "kernel arguments are limited to 4 KiB");

constexpr uint32_t kBlock = 32;  // elements of a state in 8 bits that share a scale
// A workgroup of the AdamW step: its threads, how many vectors of four elements a lane has, and how many wavefronts a SIMD
// may hold (a bound in the kernel's own attributes).
struct AdamwShape {
  uint32_t threads, vectors, waves;
  constexpr uint32_t tile() const { return threads * vectors * 4; }
};
// In fp32 four streams are read and three written, and what bounds them is how HBM mixes these: it likes few bytes in
// flight. us over 1.0 G elements / over 27 M with clipping and a copy, of which a part stays in the last-level cache: one
// wavefront of 256 elements at a time, 3 to a SIMD 4411 / 142 (6.4 TB/s), 4 4500 / 140, 8 4619 / 143; 128 threads 4655 / 139;
// 256 threads 4897 / 139; two vectors to a lane 5143 / 142. States in 8 bits have arithmetic to hide, 78 instructions for
// an element: 256 threads x 2 130, x 1 132, 64 x 2 132 us over 27 M with clipping and values read out.
constexpr AdamwShape adamw_shape(bool eight) { return eight ? AdamwShape{256, 2, 8} : AdamwShape{64, 1, 3}; }
constexpr uint32_t kAdamwWords = 400;
struct AdamwLaunch {
  float beta1, beta2, one_minus_beta1, one_minus_beta2;
  float decay;          // 1 - lr * weight_decay
  float step_size;      // lr / (1 - beta1^t)
  float root_scale;     // 1 / sqrt(1 - beta2^t)
  float eps, grad_scale, max_norm;
  const float* squared_norm;
  uint32_t seed, first_item, stochastic;
  uint32_t n_items, n_tiles;
  // An item takes the words that it needs: five pointers or six with a copy, of states in 8 bits two more for the scales. So
  // a launch has room for 80, 66, 57 or 50 of them (a launch costs the host about 3 us).
  uint32_t words_per_item;
  uint32_t first_tile[kAdamwWords / 5 + 1];
  uint64_t words[kAdamwWords];

  static constexpr uint32_t words_of(bool eight, bool copies) { return 5 + copies + 2 * eight; }
  void set(uint32_t k, const odc_adamw_item& item) {
    uint64_t* w = words + k * words_per_item;
    const void* const pointers[] = {item.param, item.grad, item.exp_avg, item.exp_avg_sq};
    *w++ = item.elems;
    for (const void* p : pointers) *w++ = (uint64_t)(uintptr_t)p;
    const bool eight = words_per_item >= 7, copies = words_per_item % 2 == 0;
    if (eight) *w++ = (uint64_t)(uintptr_t)item.exp_avg_scale, *w++ = (uint64_t)(uintptr_t)item.exp_avg_sq_scale;
    if (copies) *w++ = (uint64_t)(uintptr_t)item.copy;
  }
};
static_assert(sizeof(AdamwLaunch) <= 3900, "kernel arguments are limited to 4 KiB");

}  // namespace odc_ops_launch

namespace odc_ops_device {

// Each returns 0 or a hipError_t.
int launch_norm_forward(const odc_norm_forward& call, const odc_ops_launch::NormForwardPlan& plan, void* stream);
int launch_norm_backward(const odc_norm_backward& call, const odc_ops_launch::NormBackwardPlan& plan, void* stream);
int launch_squared_norm(int32_t dtype, bool stream_past_caches, const odc_ops_launch::SquaredNormLaunch& launch, uint32_t blocks, double* partials, void* stream);
int launch_squared_norm_total(const double* partials, uint32_t n, float* result, void* stream);
int launch_adamw(int32_t param, int32_t grad, int32_t copy, int32_t state_bits, bool stream_past_caches, const odc_ops_launch::AdamwLaunch& launch,
                 void* stream);
int launch_dequantize(const void* codes, const void* scales, void* values, uint64_t elems, int32_t dtype, void* stream);
const char* error_string(int code);

}  // namespace odc_ops_device

#endif  // ODC_OPS_LAUNCH_H_
