// odc_norm_kernels.hip — layer norm forward and backward for gfx950.
//
// y = z w + b with z = (x - mean) / sqrt(var + eps), of a row at a time; backward, with h = dy w:
// dx = (h - mean(h) - z mean(h z)) / sqrt(var + eps), and dw = sum dy z, db = sum dy over the rows. About 8 and 17
// instructions for an element, so HBM bounds them where they are not too short: x is read and y written once (4 bytes for an element of
// 16 bits), dy and x read and dx written once (6), 2 more each way with a residual.
#include "odc_ops_device.h"
#include "odc_ops_launch.h"

namespace odc_ops_device {
namespace {

using namespace odc_ops_launch;

// ------------------------------------------------------------------------------------------------
// rows in registers
// ------------------------------------------------------------------------------------------------
// kElems neighbouring elements of a row from element i on; what lies behind the row's end is zero, and neither read
// nor written. kAccess says how:
// kPlainRows: at any alignment. A piece that reaches over the row's end is read so that it ends with the row, which needs
// no branch around the loads, and the elements in front of its own are taken for zeros (rows have a whole piece at least);
// kBufferRows: rows start at multiples of 16 bytes and end with a whole piece, and all lanes agree on the row. It is a
// buffer of its own to the hardware, whose bounds check takes the place of clamped addresses (16384 x 4096 bf16 in
// rows 4104 apart: backward 79 us, 109 by plain accesses to the same rows 2 bytes on; forward level, 54 and 52);
// kStreamRows: the same, nontemporal.
template <int kElems, class T, RowAccess kAccess>
struct Piece {
  static constexpr int kVectors = kElems / Vector<T>::kElems;
  static constexpr int kPolicy = kAccess == kStreamRows ? 2 : 0;  // of a buffer access: nontemporal
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  typename Vector<T>::type v[kVectors];

  __device__ __forceinline__ void load(const T* row, uint32_t i, uint32_t width) {
    if constexpr (kAccess != kPlainRows) {
      const auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(row), 0, width * sizeof(T), 0x00027000);
#pragma unroll
      for (int k = 0; k < kVectors; ++k)
        v[k] = __builtin_bit_cast(typename Vector<T>::type, (u32x4)__builtin_amdgcn_raw_buffer_load_b128(buffer, i * sizeof(T) + k * 16, 0, kPolicy));
    } else if (width) {
      const uint32_t from = min(i, width - kElems);
#pragma unroll
      for (int k = 0; k < kVectors; ++k) v[k] = *reinterpret_cast<const typename Vector<T>::unaligned*>(row + from + k * Vector<T>::kElems);
    } else {
#pragma unroll
      for (int e = 0; e < kElems; ++e) set(e, (T)0.0f);
    }
  }
  // Behind load: element e of the piece is element i + e of the row.
  __device__ __forceinline__ void settle(uint32_t i, uint32_t width) {
    if constexpr (kAccess == kPlainRows) {
      const uint32_t over = i - min(i, width - kElems);  // elements in front of the piece's own
      if (over) {
        // one after the other, each by the one `over` places on
#pragma unroll
        for (int e = 0; e < kElems; ++e) {
          T x = (T)0.0f;
#pragma unroll
          for (int f = e; f < kElems; ++f)
            if ((uint32_t)f == e + over) x = v[f / Vector<T>::kElems][f % Vector<T>::kElems];
          set(e, x);
        }
      }
    }
  }
  __device__ __forceinline__ void store(T* row, uint32_t i, uint32_t width) const {
    if constexpr (kAccess != kPlainRows) {
      const auto buffer = __builtin_amdgcn_make_buffer_rsrc(row, 0, width * sizeof(T), 0x00027000);
#pragma unroll
      for (int k = 0; k < kVectors; ++k)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v[k]), buffer, i * sizeof(T) + k * 16, 0, kPolicy);
    } else if (i + kElems <= width) {
#pragma unroll
      for (int k = 0; k < kVectors; ++k) *reinterpret_cast<typename Vector<T>::unaligned*>(row + i + k * Vector<T>::kElems) = v[k];
    } else {
#pragma unroll
      for (int e = 0; e < kElems; ++e)
        if (i + e < width) row[i + e] = v[e / Vector<T>::kElems][e % Vector<T>::kElems];
    }
  }
  __device__ __forceinline__ float operator[](int e) const { return to_float(v[e / Vector<T>::kElems][e % Vector<T>::kElems]); }
  __device__ __forceinline__ void set(int e, T x) { v[e / Vector<T>::kElems][e % Vector<T>::kElems] = x; }
  // What was computed from it so far is forgotten: the compiler would keep the converted values over a barrier, in
  // twice the registers, where converting them again costs an instruction each.
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int k = 0; k < kVectors; ++k) asm("" : "+v"(reinterpret_cast<u32x4&>(v[k])));
  }
};

// The same access for what stays in the caches: weights, which every workgroup reads.
constexpr RowAccess kept(RowAccess access) { return access == kStreamRows ? kBufferRows : access; }

// Which of a workgroup's rows a thread works on: the same for all of a wavefront where a row takes one or more, which
// keeps the rows' addresses in scalar registers.
template <int kLanes>
__device__ __forceinline__ uint32_t row_slot() {
  const uint32_t slot = threadIdx.x / kLanes;
  return kLanes >= 64 ? __builtin_amdgcn_readfirstlane(slot) : slot;
}

// Whether any lane of this wavefront has elements of the row in its vector k, where lanes have more than one: in rows just
// above a power of two most of the second vectors are empty. (16384 x 4104 bf16 forward 70 -> 56 us. Asked for single
// vectors too, where whole wavefronts may be empty, it costs the backward pass over 16384 x 4096 3 of 74.)
template <int kLanes, int kVectors, int kElems>
__device__ __forceinline__ bool any_inside(int k, uint32_t width) {
  if constexpr (kLanes <= 64 || kVectors == 1) return true;
  return (k * kLanes + __builtin_amdgcn_readfirstlane(threadIdx.x % kLanes)) * kElems < width;
}

// The sums of kValues values over the lanes of a row. More than a wavefront's meet in LDS: `scratch` has kValues floats
// for every wavefront, and the caller alternates between two of them, so that one barrier is enough.
template <int kLanes, int kValues>
__device__ __forceinline__ void row_sums(float (&x)[kValues], float* scratch) {
#pragma unroll
  for (int v = 0; v < kValues; ++v) x[v] = sum_lanes<(kLanes < 64 ? kLanes : 64)>(x[v]);
  if constexpr (kLanes > 64) {
    const uint32_t wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 0) {
#pragma unroll
      for (int v = 0; v < kValues; ++v) scratch[wave * kValues + v] = x[v];
    }
    __syncthreads();
    constexpr int kWaves = kLanes / 64;  // neighbouring lanes take one wavefront's sums each
    const float* mine = scratch + (wave / kWaves * kWaves + threadIdx.x % kWaves) * kValues;
#pragma unroll
    for (int v = 0; v < kValues; ++v) x[v] = sum_lanes<kWaves>(mine[v]);
  }
}

// A row is read once and stays in the registers of its lanes: mean, then the variance about it (not the difference of two large
// sums) and what the mean's roundings left, then the output. Weights stay in registers for all rows of a workgroup; the next row is
// on its way meanwhile: 64 KiB in flight on a CU. 16384 x 4096 bf16 44 us (6.1 TB/s), 4096 x 4096 13.4 (5.0),
// 16384 x 14336 with a residual 323 (5.8 TB/s), 2048 x 256 fp32 3.0.
template <class T, class W, int kLanes, int kVectors, RowAccess kAccess, bool kAdd>
__global__ __launch_bounds__(kLanes > (int)kForwardThreads ? kLanes : (int)kForwardThreads) void norm_forward_kernel(odc_norm_forward c) {
  constexpr int kThreads = kLanes > (int)kForwardThreads ? kLanes : (int)kForwardThreads;
  constexpr int kElems = Vector<T>::kElems;
  __shared__ float scratch[2][2 * kThreads / 64];
  const uint32_t width = (uint32_t)c.width, lane = threadIdx.x % kLanes;
  const float per_element = 1.0f / (float)width;
  Piece<kElems, W, kept(kAccess)> weight[kVectors], bias[kVectors];
#pragma unroll
  for (int k = 0; k < kVectors; ++k) {
    const uint32_t i = (k * kLanes + lane) * kElems;
    if (c.weight) {
      weight[k].load(static_cast<const W*>(c.weight), i, width);
      weight[k].settle(i, width);
    } else {
#pragma unroll
      for (int e = 0; e < kElems; ++e) weight[k].set(e, (W)1.0f);
    }
    if (c.bias) {
      bias[k].load(static_cast<const W*>(c.bias), i, width);
      bias[k].settle(i, width);
    } else {
#pragma unroll
      for (int e = 0; e < kElems; ++e) bias[k].set(e, (W)0.0f);
    }
  }
  constexpr uint32_t kRows = kThreads / kLanes;  // at once
  uint64_t row = (uint64_t)blockIdx.x * kRows + row_slot<kLanes>();
  Piece<kElems, T, kAccess> x[kVectors], r[kVectors];
  const auto load = [&](Piece<kElems, T, kAccess>(&piece)[kVectors], const void* rows, uint64_t stride) {
#pragma unroll
    for (int k = 0; k < kVectors; ++k) piece[k].load(static_cast<const T*>(rows) + row * stride, (k * kLanes + lane) * kElems, row < c.rows ? width : 0);
  };
  const auto load_row = [&](Piece<kElems, T, kAccess>(&piece)[kVectors]) {
    load(piece, c.input, c.input_stride);
    if constexpr (kAdd) load(r, c.residual, c.residual_stride);
  };
  constexpr bool kAhead = kVectors <= 2;  // with more the registers are full
  if constexpr (kAhead) load_row(x);
  while (row < c.rows) {
    if constexpr (!kAhead) load_row(x);
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      x[k].settle((k * kLanes + lane) * kElems, width);
      if constexpr (kAdd) r[k].settle((k * kLanes + lane) * kElems, width);
    }
    if constexpr (kAdd) {
#pragma unroll
      for (int k = 0; k < kVectors; ++k) {
        if (!any_inside<kLanes, kVectors, kElems>(k, width)) continue;
#pragma unroll
        for (int e = 0; e < kElems; ++e) x[k].set(e, from_float<T>(x[k][e] + r[k][e]));
        x[k].store(static_cast<T*>(c.total) + row * c.width, (k * kLanes + lane) * kElems, width);
      }
    }
    float sum[1] = {};
#pragma unroll
    for (int k = 0; k < kVectors; ++k)
#pragma unroll
      for (int e = 0; e < kElems; ++e) sum[0] += x[k][e];
    const uint64_t here = row;
    Piece<kElems, T, kAccess> next[kVectors];
    row += (uint64_t)gridDim.x * kRows;  // the next row is on its way while this one's sums are made
    if constexpr (kAhead) load_row(next);
    row_sums<kLanes>(sum, scratch[0]);
    const float about = sum[0] / (float)width;  // the mean, but for the sum's roundings
#pragma unroll
    for (int k = 0; k < kVectors; ++k) x[k].forget();
    // about it: the squares, and in fp32 what the elements differ by on the average, which is what `about` is off by. (Sums of up to
    // 32768 values of 8 or 11 bits have hardly a rounding; there the second sum cost 4096 x 4096 bf16 5 % of 12.8 us.)
    constexpr bool kCorrected = sizeof(T) == 4;
    float moments[1 + kCorrected] = {};
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      if (!any_inside<kLanes, kVectors, kElems>(k, width)) continue;
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        const float d = (k * kLanes + lane) * kElems + (kAccess != kPlainRows ? 0 : e) < width ? x[k][e] - about : 0.0f;
        moments[0] += d * d;
        if constexpr (kCorrected) moments[1] += d;
      }
    }
    row_sums<kLanes>(moments, scratch[1]);
    float mean = about, variance = moments[0] * per_element;
    if constexpr (kCorrected) {
      const float off = moments[1] * per_element;
      mean += off;
      if (variance < INFINITY) variance = fmaxf(variance - off * off, 0.0f);
    }
    const float rstd = 1.0f / sqrtf(variance + c.eps);
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      if (any_inside<kLanes, kVectors, kElems>(k, width)) {
        x[k].forget();
#pragma unroll
        for (int e = 0; e < kElems; ++e) x[k].set(e, from_float<T>((x[k][e] - mean) * rstd * weight[k][e] + bias[k][e]));
        x[k].store(static_cast<T*>(c.output) + here * c.width, (k * kLanes + lane) * kElems, width);
      }
      if constexpr (kAhead) x[k] = next[k];
    }
    if (lane == 0) {
      if (c.mean) c.mean[here] = mean;
      if (c.rstd) c.rstd[here] = rstd;
    }
  }
}

// A workgroup passes over rows blockIdx.x, + gridDim.x, ... (kThreads / kLanes of them at once), writes their
// grad_input and keeps the sums for weight and bias of its lanes' columns in registers; at the end the rows that it had
// at once are added in LDS, upper half onto lower half, and go to its row of the workspace.
// 16384 x 4096 bf16 74 us (5.4 TB/s), 4096 x 4096 25 (4.0: 16 rows to a workgroup, start and end are a third of it), 16384 x
// 14336 with a residual 326 (5.8).
template <class T, class W, int kLanes, int kVectors, RowAccess kAccess>
__global__ __launch_bounds__(kBackwardThreads) void norm_backward_kernel(odc_norm_backward c) {
  constexpr int kThreads = kBackwardThreads, kElems = Vector<T>::kElems, kRows = kThreads / kLanes;
  constexpr int kSums = 2 * kVectors * kElems;  // of a thread
  __shared__ float scratch[2][2 * kThreads / 64];
  __shared__ float upper[kRows > 1 ? kThreads / 2 * kSums : 1];
  const uint32_t width = (uint32_t)c.width, lane = threadIdx.x % kLanes, slot = row_slot<kLanes>();
  const float per_element = 1.0f / (float)width;
  const bool sums = c.grad_weight || c.grad_bias;
  // The weights of a lane's columns stay in registers, or, where the sums and the rows need these, in LDS: every lane
  // puts its own there.
  constexpr bool kWeightInLds = kVectors > 1;
  typedef Piece<kElems, W, kept(kAccess)> Weight;
  __shared__ typename Vector<W>::type weights[kWeightInLds ? kVectors * Weight::kVectors * kThreads : 1];
  Weight weight_here[kWeightInLds ? 1 : kVectors];
  float dw[kVectors][kElems] = {}, db[kVectors][kElems] = {};
#pragma unroll
  for (int k = 0; k < kVectors; ++k) {
    Weight w;
    if (c.weight) {
      w.load(static_cast<const W*>(c.weight), (k * kLanes + lane) * kElems, width);
      w.settle((k * kLanes + lane) * kElems, width);
    } else {
#pragma unroll
      for (int e = 0; e < kElems; ++e) w.set(e, (W)1.0f);
    }
    if constexpr (kWeightInLds) {
#pragma unroll
      for (int v = 0; v < Weight::kVectors; ++v) weights[(k * Weight::kVectors + v) * kThreads + threadIdx.x] = w.v[v];
    } else {
      weight_here[k] = w;
    }
  }
  const auto weight = [&](int k) {
    if constexpr (!kWeightInLds) return weight_here[k];
    Weight w;
#pragma unroll
    for (int v = 0; v < Weight::kVectors; ++v) w.v[v] = weights[(k * Weight::kVectors + v) * kThreads + threadIdx.x];
    return w;
  };
  int parity = 0;
  struct Row {
    Piece<kElems, T, kAccess> x[kVectors], dy[kVectors], dt[kVectors];
    float mean, rstd;
  };
  const auto load = [&](Piece<kElems, T, kAccess>(&piece)[kVectors], const void* rows, uint64_t stride, uint64_t row) {
#pragma unroll
    for (int k = 0; k < kVectors; ++k)
      piece[k].load(static_cast<const T*>(rows) + row * stride, (k * kLanes + lane) * kElems, row < c.rows && rows ? width : 0);
  };
  const auto load_total = [&](Row& r, uint64_t row) {
    if (c.grad_input) load(r.dt, c.grad_total, c.grad_total_stride, row);
  };
  const auto load_row = [&](Row& r, uint64_t row) {
    load(r.dy, c.grad_output, c.grad_output_stride, row);
    load(r.x, c.normalised, c.normalised_stride, row);
    r.mean = row < c.rows ? c.mean[row] : 0;
    r.rstd = row < c.rows ? c.rstd[row] : 0;
  };
  // Rows on their way while one's sums are made, as far as registers go: with 16 wavefronts on a CU, 32 bytes to a lane and
  // row, one row ahead is half of what keeps HBM busy.
  constexpr int kAhead = kVectors == 1 ? kRowsAhead : kVectors == 2 && kAccess != kPlainRows ? 1 : 0;
  constexpr bool kTotalAhead = kVectors == 1;
  const uint64_t step = (uint64_t)gridDim.x * kRows;
  Row ring[kAhead + 1];
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    load_row(ring[a], (uint64_t)blockIdx.x * kRows + slot + a * step);
    if constexpr (kTotalAhead) load_total(ring[a], (uint64_t)blockIdx.x * kRows + slot + a * step);
  }
  // every thread makes the same number of rounds: there are barriers in them
  for (uint64_t first = (uint64_t)blockIdx.x * kRows; first < c.rows; first += step, parity ^= 1) {
    const uint64_t row = first + slot;
    const bool mine = row < c.rows;
    Row& r = ring[0];
    if constexpr (kAhead == 0) load_row(r, row);
    float row_sum[2] = {};
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      if (!any_inside<kLanes, kVectors, kElems>(k, width)) continue;
      r.x[k].settle((k * kLanes + lane) * kElems, width);
      r.dy[k].settle((k * kLanes + lane) * kElems, mine ? width : 0);
      const Weight w = weight(k);
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        const float z = (r.x[k][e] - r.mean) * r.rstd, g = r.dy[k][e];  // behind the row's end g is zero and z of no account
        const float h = g * w[e];
        row_sum[0] += h;
        row_sum[1] += h * z;
        dw[k][e] += g * z;
        db[k][e] += g;
      }
      if constexpr (kVectors > 1) __builtin_amdgcn_sched_barrier(0);  // one vector's values at a time: registers
    }
    if constexpr (!kTotalAhead) load_total(r, row);
    if constexpr (kAhead > 0) {
      load_row(ring[kAhead], row + kAhead * step);
      if constexpr (kTotalAhead) load_total(ring[kAhead], row + kAhead * step);
    }
    if (c.grad_input) {
      row_sums<kLanes>(row_sum, scratch[parity]);
      const float sum = row_sum[0] * per_element, dot = row_sum[1] * per_element;
      if (mine) {
#pragma unroll
        for (int k = 0; k < kVectors; ++k) {
          if (!any_inside<kLanes, kVectors, kElems>(k, width)) continue;
          r.x[k].forget();
          r.dy[k].forget();
          if (c.grad_total) r.dt[k].settle((k * kLanes + lane) * kElems, width);
          const Weight w = weight(k);
#pragma unroll
          for (int e = 0; e < kElems; ++e) {
            const float z = (r.x[k][e] - r.mean) * r.rstd, h = r.dy[k][e] * w[e];
            r.x[k].set(e, from_float<T>(r.rstd * (h - sum - z * dot) + r.dt[k][e]));
          }
          r.x[k].store(static_cast<T*>(c.grad_input) + row * c.width, (k * kLanes + lane) * kElems, width);
          if constexpr (kVectors > 1) __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) ring[a] = ring[a + 1];
  }
  if (!sums) return;
#pragma unroll
  for (int half = kThreads / 2; half >= kLanes; half /= 2) {
    if (threadIdx.x >= (uint32_t)half && threadIdx.x < 2u * half) {
#pragma unroll
      for (int s = 0; s < kSums; ++s) upper[s * half + threadIdx.x - half] = s % 2 ? db[s / 2 / kElems][s / 2 % kElems] : dw[s / 2 / kElems][s / 2 % kElems];
    }
    __syncthreads();
    if (threadIdx.x < (uint32_t)half) {
#pragma unroll
      for (int s = 0; s < kSums; ++s) (s % 2 ? db[s / 2 / kElems][s / 2 % kElems] : dw[s / 2 / kElems][s / 2 % kElems]) += upper[s * half + threadIdx.x];
    }
    __syncthreads();
  }
  if (threadIdx.x >= (uint32_t)kLanes) return;
  const bool alone = gridDim.x == 1;  // nothing to add, and no second launch
  W* const weight_out = static_cast<W*>(c.grad_weight);
  W* const bias_out = static_cast<W*>(c.grad_bias);
  float* const out = static_cast<float*>(c.workspace) + (uint64_t)blockIdx.x * 2 * width;
#pragma unroll
  for (int k = 0; k < kVectors; ++k)
#pragma unroll
    for (int e = 0; e < kElems; ++e) {
      const uint32_t i = (k * kLanes + lane) * kElems + e;
      if (i >= width) continue;
      if (!alone) {
        out[i] = dw[k][e];
        out[width + i] = db[k][e];
      } else {
        if (weight_out) weight_out[i] = from_float<W>(dw[k][e]);
        if (bias_out) bias_out[i] = from_float<W>(db[k][e]);
      }
    }
}

// ------------------------------------------------------------------------------------------------
// wide rows, and rows of less than a vector
// ------------------------------------------------------------------------------------------------
// kElems neighbouring elements of a row as floats, by one access where the row has that many left.
template <class T>
__device__ __forceinline__ void load_some(const T* row, uint32_t i, uint32_t width, float (&x)[Vector<T>::kElems]) {
  constexpr uint32_t kElems = Vector<T>::kElems;
  if (i + kElems <= width) {
    const typename Vector<T>::type v = *reinterpret_cast<const typename Vector<T>::unaligned*>(row + i);
#pragma unroll
    for (uint32_t e = 0; e < kElems; ++e) x[e] = to_float(v[e]);
  } else {
#pragma unroll
    for (uint32_t e = 0; e < kElems; ++e) x[e] = i + e < width ? to_float(row[i + e]) : 0.0f;
  }
}

template <class T>
__device__ __forceinline__ void store_some(T* row, uint32_t i, uint32_t width, const float (&x)[Vector<T>::kElems]) {
  constexpr uint32_t kElems = Vector<T>::kElems;
  if (i + kElems <= width) {
    typename Vector<T>::type v;
#pragma unroll
    for (uint32_t e = 0; e < kElems; ++e) v[e] = from_float<T>(x[e]);
    *reinterpret_cast<typename Vector<T>::unaligned*>(row + i) = v;
  } else {
#pragma unroll
    for (uint32_t e = 0; e < kElems; ++e)
      if (i + e < width) row[i + e] = from_float<T>(x[e]);
  }
}

// The sum of a vector's values, in pairs (exact for equal values, so that a row of one value has it for a mean; a part of a vector
// is added one by one for that). What a thread has of a row is added up in 64 bits: in 32, the 2^18 additions of the
// widest rows would leave a mean that is off by a hundredth.
template <uint32_t kElems>
__device__ __forceinline__ double sum_of(const float (&x)[kElems], bool whole = true) {
  if (!whole) {
    double sum = x[0];
#pragma unroll
    for (uint32_t e = 1; e < kElems; ++e) sum += x[e];
    return sum;
  }
  float pairs[kElems / 2];
#pragma unroll
  for (uint32_t e = 0; e < kElems / 2; ++e) pairs[e] = x[2 * e] + x[2 * e + 1];
#pragma unroll
  for (uint32_t width = kElems / 4; width; width /= 2)
#pragma unroll
    for (uint32_t e = 0; e < width; ++e) pairs[e] += pairs[e + width];
  return pairs[0];
}

// Calls body with the first elements of a thread's vectors in a row: the whole ones in a loop, whose condition is the one that
// load_some and store_some ask for, and the one that the row's end cuts behind it.
template <uint32_t kElems, class Body>
__device__ __forceinline__ void over_row(uint32_t begin, uint32_t width, Body body) {
  uint32_t i = begin;
  for (; i + kElems <= width; i += kWideThreads * kElems) body(i);
  if (i < width) body(i);
}

// The sum over a row's workgroup, in every thread. A row of less than a vector is the first thread's alone.
__device__ __forceinline__ double wide_sum(double x, bool first_alone, double* scratch) {
  if (!first_alone) return block_sum<kWideThreads>(x, scratch);
  __syncthreads();  // the last sum's readers are done
  if (threadIdx.x == 0) scratch[0] = x;
  __syncthreads();
  return scratch[0];
}

// Weights (or `otherwise` where there are none) beside the elements of a row.
template <uint32_t kElems, class W>
__device__ __forceinline__ void load_weights(const W* weights, uint32_t i, uint32_t width, float otherwise, float (&x)[kElems]) {
  if (weights && i + kElems <= width) {
    typedef W Weights __attribute__((ext_vector_type(kElems)));
    typedef Weights WeightsAnywhere __attribute__((aligned(sizeof(W))));
    const Weights v = *reinterpret_cast<const WeightsAnywhere*>(weights + i);
#pragma unroll
    for (uint32_t e = 0; e < kElems; ++e) x[e] = to_float(v[e]);
  } else {
#pragma unroll
    for (uint32_t e = 0; e < kElems; ++e) x[e] = weights && i + e < width ? to_float(weights[i + e]) : otherwise;
  }
}

// One workgroup per row, three passes over it (the second and third find it in the caches): the mean, the
// variance about that mean, the output. 4096 x 20000 fp32 with a residual 354 us (3.7 TB/s); backward, the rows and then the
// columns, 266 + 133; in bf16 123 + 69. (Rows of less than a vector: 1000000 x 4 bf16 2.8 ms, one lane of a workgroup has work.)
template <class T, class W>
__global__ __launch_bounds__(kWideThreads) void norm_forward_wide_kernel(odc_norm_forward c) {
  constexpr uint32_t kElems = Vector<T>::kElems;
  __shared__ double scratch[kWideThreads / 64];
  const uint32_t width = (uint32_t)c.width, begin = threadIdx.x * kElems;
  const W* weight = static_cast<const W*>(c.weight);
  const W* bias = static_cast<const W*>(c.bias);
  for (uint64_t row = blockIdx.x; row < c.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(c.input) + row * c.input_stride;
    const T* r = c.residual ? static_cast<const T*>(c.residual) + row * c.residual_stride : nullptr;
    T* y = static_cast<T*>(c.output) + row * c.width;
    T* total = r ? static_cast<T*>(c.total) + row * c.width : nullptr;
    double sum = 0;
    over_row<kElems>(begin, width, [&](uint32_t i) {
      float v[kElems];
      load_some(x, i, width, v);
      if (r) {
        float other[kElems];
        load_some(r, i, width, other);
#pragma unroll
        for (uint32_t e = 0; e < kElems; ++e) v[e] = to_float(from_float<T>(v[e] + other[e]));
        store_some(total, i, width, v);
      }
      sum += sum_of(v, i + kElems <= width);
    });
    const T* z = r ? total : x;  // a thread reads what it wrote itself
    const float mean = (float)(wide_sum(sum, width < kElems, scratch) / width);
    double squares = 0;
    over_row<kElems>(begin, width, [&](uint32_t i) {
      float v[kElems];
      load_some(z, i, width, v);
#pragma unroll
      for (uint32_t e = 0; e < kElems; ++e) {
        const float d = i + e < width ? v[e] - mean : 0.0f;
        v[e] = d * d;
      }
      squares += sum_of(v);
    });
    const float rstd = 1.0f / sqrtf((float)(wide_sum(squares, width < kElems, scratch) / width) + c.eps);
    over_row<kElems>(begin, width, [&](uint32_t i) {
      float v[kElems], w[kElems], b[kElems];
      load_some(z, i, width, v);
      load_weights<kElems>(weight, i, width, 1.0f, w);
      load_weights<kElems>(bias, i, width, 0.0f, b);
#pragma unroll
      for (uint32_t e = 0; e < kElems; ++e) v[e] = (v[e] - mean) * rstd * w[e] + b[e];
      store_some(y, i, width, v);
    });
    if (threadIdx.x == 0) {
      if (c.mean) c.mean[row] = mean;
      if (c.rstd) c.rstd[row] = rstd;
    }
  }
}

template <class T, class W>
__global__ __launch_bounds__(kWideThreads) void norm_backward_rows_kernel(odc_norm_backward c) {
  constexpr uint32_t kElems = Vector<T>::kElems;
  __shared__ double scratch[kWideThreads / 64];
  const uint32_t width = (uint32_t)c.width, begin = threadIdx.x * kElems;
  const W* weight = static_cast<const W*>(c.weight);
  for (uint64_t row = blockIdx.x; row < c.rows; row += gridDim.x) {
    const T* dy = static_cast<const T*>(c.grad_output) + row * c.grad_output_stride;
    const T* x = static_cast<const T*>(c.normalised) + row * c.normalised_stride;
    const T* dt = c.grad_total ? static_cast<const T*>(c.grad_total) + row * c.grad_total_stride : nullptr;
    T* dx = static_cast<T*>(c.grad_input) + row * c.width;
    const float mean = c.mean[row], rstd = c.rstd[row];
    double sums = 0, dots = 0;
    over_row<kElems>(begin, width, [&](uint32_t i) {
      float g[kElems], v[kElems], w[kElems];
      load_some(dy, i, width, g);
      load_some(x, i, width, v);
      load_weights<kElems>(weight, i, width, 1.0f, w);
#pragma unroll
      for (uint32_t e = 0; e < kElems; ++e) {
        g[e] *= w[e];
        v[e] = g[e] * ((v[e] - mean) * rstd);
      }
      sums += sum_of(g);
      dots += sum_of(v);
    });
    const float sum = (float)(wide_sum(sums, width < kElems, scratch) / width), dot = (float)(wide_sum(dots, width < kElems, scratch) / width);
    over_row<kElems>(begin, width, [&](uint32_t i) {
      float g[kElems], v[kElems], w[kElems], t[kElems] = {};
      load_some(dy, i, width, g);
      load_some(x, i, width, v);
      load_weights<kElems>(weight, i, width, 1.0f, w);
      if (dt) load_some(dt, i, width, t);
#pragma unroll
      for (uint32_t e = 0; e < kElems; ++e) v[e] = rstd * (g[e] * w[e] - sum - (v[e] - mean) * rstd * dot) + t[e];
      store_some(dx, i, width, v);
    });
  }
}

// Workgroup (tile of columns, group of rows): the sums over the group's rows, a vector of columns to a lane. Wavefront w
// takes every fourth row.
template <class T>
__global__ __launch_bounds__(kWideThreads) void norm_backward_columns_kernel(odc_norm_backward c, uint64_t rows_per_group) {
  constexpr uint32_t kWaves = kWideThreads / 64, kElems = Vector<T>::kElems, kColumns = 64 * kElems;
  __shared__ float scratch[2][kWaves][kColumns];
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, width = (uint32_t)c.width;
  const uint32_t tile = blockIdx.x * kColumns, column = tile + lane * kElems;
  const uint64_t first = blockIdx.y * rows_per_group;
  const uint64_t end = first + rows_per_group < c.rows ? first + rows_per_group : c.rows;
  float dw[kElems] = {}, db[kElems] = {};
  if (column < width) {
    for (uint64_t row = first + wave; row < end; row += kWaves) {
      float g[kElems], x[kElems];
      load_some(static_cast<const T*>(c.grad_output) + row * c.grad_output_stride, column, width, g);
      load_some(static_cast<const T*>(c.normalised) + row * c.normalised_stride, column, width, x);
      const float mean = c.mean[row], rstd = c.rstd[row];
#pragma unroll
      for (uint32_t e = 0; e < kElems; ++e) {
        dw[e] += g[e] * ((x[e] - mean) * rstd);
        db[e] += g[e];
      }
    }
  }
#pragma unroll
  for (uint32_t e = 0; e < kElems; ++e) {
    scratch[0][wave][lane * kElems + e] = dw[e];
    scratch[1][wave][lane * kElems + e] = db[e];
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < 2 * kColumns; i += kWideThreads) {
    const uint32_t which = i / kColumns, at = i % kColumns;
    if (tile + at >= width) continue;
    float sum = scratch[which][0][at];
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) sum += scratch[which][w][at];
    static_cast<float*>(c.workspace)[(2 * (uint64_t)blockIdx.y + which) * width + tile + at] = sum;
  }
}

// The sums over the groups: 32 columns of [2][width] and 32 groups at once, four columns to a thread. (Over 256 groups of
// 2 x 4096 columns 4.0 us.)
template <class W>
__global__ __launch_bounds__(256) void norm_backward_groups_kernel(odc_norm_backward c, uint32_t groups) {
  constexpr uint32_t kParts = 256 / (kGroupColumns / 4);
  __shared__ float scratch[kParts][kGroupColumns];
  const uint32_t part = threadIdx.x / (kGroupColumns / 4), quad = threadIdx.x % (kGroupColumns / 4) * 4;
  const uint64_t at = (uint64_t)blockIdx.x * kGroupColumns + quad, end = 2 * c.width;
  const float* workspace = static_cast<const float*>(c.workspace);
  float sum[4] = {};
  if (at + 4 <= end) {
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll 8
    for (uint32_t g = part; g < groups; g += kParts) {
      const f4 v = *reinterpret_cast<const f4*>(workspace + g * end + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += v[e];
    }
  } else {
    for (uint32_t g = part; g < groups; g += kParts)
      for (int e = 0; e < 4; ++e)
        if (at + e < end) sum[e] += workspace[g * end + at + e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) scratch[part][quad + e] = sum[e];
  __syncthreads();
  const uint64_t column = (uint64_t)blockIdx.x * kGroupColumns + threadIdx.x;
  if (threadIdx.x < kGroupColumns && column < end) {
    float all = scratch[0][threadIdx.x];
#pragma unroll
    for (uint32_t p = 1; p < kParts; ++p) all += scratch[p][threadIdx.x];
    W* out = static_cast<W*>(column < c.width ? c.grad_weight : c.grad_bias);
    if (out) out[column < c.width ? column : column - c.width] = from_float<W>(all);
  }
}

// ------------------------------------------------------------------------------------------------
// launches
// ------------------------------------------------------------------------------------------------
// Calls body with a value of the element types' own.
template <class Body>
int with_types(int32_t dtype, int32_t weight_dtype, Body body) {
  if (dtype == ODC_OPS_F32) return body(float(), float());
  if (dtype == ODC_OPS_BF16) return weight_dtype == ODC_OPS_F32 ? body(bf16(), float()) : body(bf16(), bf16());
  return weight_dtype == ODC_OPS_F32 ? body(f16(), float()) : body(f16(), f16());
}

template <uint32_t n>
struct Number {
  static constexpr uint32_t value = n;
};

// Calls body with the shape's lanes and vectors as types; shapes[kAt] and those behind it.
template <const auto& kShapes, size_t kAt = 0, class Body>
void with_shape(NormShape shape, Body body) {
  constexpr NormShape s = kShapes[kAt];
  if (shape.lanes == s.lanes && shape.vectors == s.vectors) return body(Number<s.lanes>(), Number<s.vectors>());
  if constexpr (kAt + 1 < sizeof(kShapes) / sizeof(NormShape)) with_shape<kShapes, kAt + 1>(shape, body);
}

template <class Body>
void with_truth(bool truth, Body body) {
  if (truth) body(Number<1>());
  else body(Number<0>());
}

// Rows that share a wavefront are no buffers (access_of in odc_ops_host.cpp does not say so either).
template <int kLanes, class Body>
void with_access(RowAccess access, Body body) {
  if constexpr (kLanes >= 64) {
    if (access == kStreamRows) return body(Number<kStreamRows>());
    if (access == kBufferRows) return body(Number<kBufferRows>());
  }
  body(Number<kPlainRows>());
}

}  // namespace

int launch_norm_forward(const odc_norm_forward& call, const NormForwardPlan& plan, void* stream) {
  return with_types(call.dtype, call.weight_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    if (!plan.shape.lanes) return launch(norm_forward_wide_kernel<T, W>, plan.blocks, kWideThreads, stream, call);
    int status = (int)hipErrorInvalidDeviceFunction;
    with_shape<kForwardShapes>(plan.shape, [&](auto lanes, auto vectors) {
      constexpr int kLanes = decltype(lanes)::value, kVectors = decltype(vectors)::value;
      constexpr int kThreads = kLanes > (int)kForwardThreads ? kLanes : (int)kForwardThreads;
      with_access<kLanes>(plan.access, [&](auto access) {
        with_truth(call.residual != nullptr, [&](auto add) {
          status = launch(norm_forward_kernel<T, W, kLanes, kVectors, (RowAccess)decltype(access)::value, decltype(add)::value>, plan.blocks, kThreads,
                          stream, call);
        });
      });
    });
    return status;
  });
}

int launch_norm_backward(const odc_norm_backward& call, const NormBackwardPlan& plan, void* stream) {
  return with_types(call.dtype, call.weight_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    const bool sums = call.grad_weight || call.grad_bias;
    int status = 0;
    if (plan.shape.lanes && plan.groups) {
      status = (int)hipErrorInvalidDeviceFunction;
      const auto launch_rows = [&](auto lanes, auto vectors) {
        constexpr int kLanes = decltype(lanes)::value, kVectors = decltype(vectors)::value;
        with_access<kLanes>(plan.access, [&](auto access) {
          status = launch(norm_backward_kernel<T, W, kLanes, kVectors, (RowAccess)decltype(access)::value>, plan.groups, kBackwardThreads, stream, call);
        });
      };
      if constexpr (sizeof(T) == 4) with_shape<kBackwardShapes32>(plan.shape, launch_rows);
      else with_shape<kBackwardShapes16>(plan.shape, launch_rows);
    } else if (plan.groups) {
      if (call.grad_input) status = launch(norm_backward_rows_kernel<T, W>, plan.row_blocks, kWideThreads, stream, call);
      constexpr uint32_t kColumns = 64 * Vector<T>::kElems;
      const uint32_t tiles = (uint32_t)((call.width + kColumns - 1) / kColumns);
      if (!status && sums) status = launch(norm_backward_columns_kernel<T>, dim3(tiles, plan.groups), kWideThreads, stream, call, plan.rows_per_group);
    }
    if (!status && sums && !plan.one_launch()) {
      const uint32_t blocks = (uint32_t)((2 * call.width + kGroupColumns - 1) / kGroupColumns);
      status = launch(norm_backward_groups_kernel<W>, blocks, 256, stream, call, plan.groups);
    }
    return status;
  });
}

const char* error_string(int code) { return hipGetErrorString((hipError_t)code); }

}  // namespace odc_ops_device
