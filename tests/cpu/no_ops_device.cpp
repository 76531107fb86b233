// An odc_ops_device (odc_amd/csrc/odc_ops_launch.h) for a machine without a GPU, and checks of the host side of
// libodc_ops.so on it: what is refused, what launches are planned, that every tile of a list has its item and
// every item its tiles. Built by g++ under AddressSanitizer and UBSan with odc_amd/csrc/odc_ops_host.cpp.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "odc_ops.h"
#include "odc_ops_launch.h"

using namespace odc_ops_launch;

namespace {
struct Seen {
  int norm_forward = 0, norm_backward = 0, totals = 0, dequantize = 0;
  std::vector<SquaredNormLaunch> squared;
  std::vector<uint32_t> squared_blocks;
  std::vector<double*> squared_partials;
  std::vector<AdamwLaunch> adamw;
  uint32_t total_partials = 0;
} seen;
int answer = 0;
}  // namespace

namespace odc_ops_device {
int launch_norm_forward(const odc_norm_forward&, const NormForwardPlan&, void*) { return ++seen.norm_forward, answer; }
int launch_norm_backward(const odc_norm_backward&, const NormBackwardPlan&, void*) { return ++seen.norm_backward, answer; }
int launch_squared_norm(int32_t, bool, const SquaredNormLaunch& launch, uint32_t blocks, double* partials, void*) {
  seen.squared.push_back(launch);
  seen.squared_blocks.push_back(blocks);
  seen.squared_partials.push_back(partials);
  return answer;
}
int launch_squared_norm_total(const double*, uint32_t n, float*, void*) {
  ++seen.totals;
  seen.total_partials = n;
  return answer;
}
int launch_adamw(int32_t, int32_t, int32_t, int32_t, bool, const AdamwLaunch& launch, void*) { return seen.adamw.push_back(launch), answer; }
int launch_dequantize(const void*, const void*, void*, uint64_t, int32_t, void*) { return ++seen.dequantize, answer; }
const char* error_string(int) { return "no device"; }
}  // namespace odc_ops_device

#define CHECK(cond)                                                                                 \
  do {                                                                                              \
    if (!(cond)) {                                                                                  \
      fprintf(stderr, "%s:%d: %s (%s)\n", __FILE__, __LINE__, #cond, odc_ops_last_error());          \
      exit(1);                                                                                      \
    }                                                                                               \
  } while (0)

namespace {

// Made-up device addresses: nothing here reads through them.
void* at(uintptr_t address) { return reinterpret_cast<void*>(address); }

void check_item(const AdamwLaunch& launch, uint32_t i, const odc_adamw_item& item) {
  const uint64_t* w = launch.words + i * launch.words_per_item;
  const auto is = [](uint64_t word, const void* p) { return word == (uint64_t)(uintptr_t)p; };
  CHECK((i + 1) * launch.words_per_item <= kAdamwWords);
  CHECK(w[0] == item.elems && is(w[1], item.param) && is(w[2], item.grad) && is(w[3], item.exp_avg) && is(w[4], item.exp_avg_sq));
  const uint32_t scales = launch.words_per_item >= 7 ? 2 : 0;
  CHECK(!scales || (is(w[5], item.exp_avg_scale) && is(w[6], item.exp_avg_sq_scale)));
  CHECK(launch.words_per_item == 5 + scales + (item.copy != nullptr) && (!item.copy || is(w[5 + scales], item.copy)));
}
void check_item(const SquaredNormLaunch& launch, uint32_t i, const odc_span_item& item) {
  const uint64_t tiles = launch.first_tile[i + 1] - launch.first_tile[i], last = launch.places[i] & 0xFFFF;
  CHECK(launch.places[i] >> 16 == (uint64_t)(uintptr_t)item.data && (tiles ? (tiles - 1) * kNormTile + last : 0) == item.elems);
}

// The tables of a list's launches: every item in order, with as many tiles as its elements need.
template <class Launch, class Item>
void check_tables(const std::vector<Launch>& launches, const std::vector<Item>& items, uint32_t tile) {
  size_t k = 0;
  for (const Launch& launch : launches) {
    CHECK(launch.n_tiles > 0 && launch.first_tile[0] == 0 && launch.first_tile[launch.n_items] == launch.n_tiles);
    for (uint32_t i = 0; i < launch.n_items; ++i, ++k) {
      check_item(launch, i, items[k]);
      CHECK(launch.first_tile[i + 1] - launch.first_tile[i] == (items[k].elems + tile - 1) / tile);
    }
  }
  for (; k < items.size(); ++k) CHECK(items[k].elems == 0);
}

void check_layer_norm() {
  odc_norm_forward f = {};
  f.rows = 10, f.width = 100, f.input_stride = 100, f.dtype = ODC_OPS_BF16, f.weight_dtype = ODC_OPS_F32, f.eps = 1e-5f;
  f.input = at(0x1000), f.output = at(0x2000);
  CHECK(odc_layer_norm(&f, nullptr) == ODC_OPS_OK && seen.norm_forward == 1);
  const auto refused = [&](auto change) {
    odc_norm_forward g = f;
    change(g);
    const int before = seen.norm_forward, rc = odc_layer_norm(&g, nullptr);
    CHECK(rc < 0 && seen.norm_forward == before && *odc_ops_last_error());
  };
  CHECK(odc_layer_norm(nullptr, nullptr) == ODC_OPS_ERR_INVALID);
  refused([](auto& g) { g.input = nullptr; });
  refused([](auto& g) { g.output = nullptr; });
  refused([](auto& g) { g.input = at(0x1001); });
  refused([](auto& g) { g.weight = at(0x1002); });
  refused([](auto& g) { g.mean = reinterpret_cast<float*>(at(0x1002)); });
  refused([](auto& g) { g.residual = at(0x4000); });  // without total
  refused([](auto& g) { g.total = at(0x4000); });     // without residual
  refused([](auto& g) { g.dtype = 3; });
  refused([](auto& g) { g.dtype = ODC_OPS_NONE; });
  refused([](auto& g) { g.weight_dtype = ODC_OPS_F16; });
  refused([](auto& g) { g.width = g.input_stride = (uint64_t(1) << 26) + 1; });
  refused([](auto& g) { g.rows = uint64_t(1) << 58; });
  refused([](auto& g) { g.input_stride = uint64_t(1) << 58; });
  f.rows = 0;
  f.input = nullptr;
  CHECK(odc_layer_norm(&f, nullptr) == ODC_OPS_OK && seen.norm_forward == 1);

  odc_norm_backward b = {};
  b.rows = 1000, b.width = 100, b.grad_output_stride = b.normalised_stride = b.grad_total_stride = 100;
  b.dtype = ODC_OPS_F32, b.weight_dtype = ODC_OPS_F32;
  b.grad_output = at(0x1000), b.normalised = at(0x2000), b.grad_input = at(0x3000), b.grad_weight = at(0x4000);
  b.mean = b.rstd = static_cast<float*>(at(0x5000));
  b.workspace = at(0x6000);
  b.workspace_bytes = odc_layer_norm_backward_workspace(b.rows, b.width, b.dtype);
  CHECK(b.workspace_bytes >= 2 * 100 * 4 && odc_layer_norm_backward_workspace(0, 100, b.dtype) == 0);
  CHECK(odc_layer_norm_backward(&b, nullptr) == ODC_OPS_OK && seen.norm_backward == 1);
  const auto refused_back = [&](auto change) {
    odc_norm_backward g = b;
    change(g);
    const int before = seen.norm_backward, rc = odc_layer_norm_backward(&g, nullptr);
    CHECK(rc < 0 && seen.norm_backward == before);
  };
  refused_back([](auto& g) { g.grad_output = nullptr; });
  refused_back([](auto& g) { g.normalised = at(0x2001); });
  refused_back([](auto& g) { g.mean = nullptr; });
  refused_back([](auto& g) { g.workspace = nullptr; });
  refused_back([](auto& g) { g.workspace = at(0x6004); });
  refused_back([](auto& g) { --g.workspace_bytes; });
  refused_back([](auto& g) { g.grad_bias = at(0x4001); });
  refused_back([](auto& g) { g.grad_total = at(0x4001); });
  b.grad_weight = nullptr;
  b.workspace = nullptr;  // not needed for grad_input alone
  CHECK(odc_layer_norm_backward(&b, nullptr) == ODC_OPS_OK && seen.norm_backward == 2);
  // plans: groups of rows that cover all of them, none without rows
  for (uint64_t rows : {1ull, 2ull, 3ull, 255ull, 256ull, 257ull, 1000ull, 4096ull, 65537ull, 10000000ull})
    for (uint64_t width : {1ull, 64ull, 256ull, 1001ull, 4096ull, 14336ull, 100000ull})
      for (int32_t dtype : {ODC_OPS_BF16, ODC_OPS_F32})
        CHECK(odc_layer_norm_backward_workspace(rows, width, dtype) % (2 * width * 4) == 0);
}

void check_lists() {
  std::vector<std::vector<uint64_t>> lists = {{1}, {0}, {0, 0, 5, 0}, {}, {100000000}, {uint64_t(5) << 30, 7}};
  lists.emplace_back(500, 3000);
  lists.emplace_back(161, 1);
  lists.emplace_back();
  for (int k = 0; k < 300; ++k) lists.back().push_back((uint64_t)(k * 7919 % 100000) * (k % 7 != 0));
  for (const auto& sizes : lists) {
    std::vector<odc_span_item> spans;
    std::vector<odc_adamw_item> items;
    for (uint64_t n : sizes) {
      spans.push_back({n ? at(0x1000) : nullptr, n});
      items.push_back({at(0x1000), at(0x2000), at(0x3000), at(0x4000), at(0x5001), at(0x6001), nullptr, n});
    }
    seen = Seen();
    const uint64_t bytes = odc_squared_norm_workspace(spans.data(), (uint32_t)spans.size(), ODC_OPS_BF16);
    std::vector<double> workspace(bytes / sizeof(double) + 1);
    float result;
    CHECK(odc_squared_norm(spans.data(), (uint32_t)spans.size(), ODC_OPS_BF16, workspace.data(), bytes, &result, nullptr) == ODC_OPS_OK);
    check_tables(seen.squared, spans, kNormTile);
    CHECK(seen.totals == 1 && seen.total_partials * sizeof(double) <= bytes);
    uint64_t done = 0;
    for (size_t k = 0; k < seen.squared.size(); ++k) {
      CHECK(seen.squared_partials[k] == workspace.data() + done && seen.squared_blocks[k] > 0 && seen.squared_blocks[k] <= seen.squared[k].n_tiles);
      done += seen.squared_blocks[k];
    }
    if (bytes) CHECK(odc_squared_norm(spans.data(), (uint32_t)spans.size(), ODC_OPS_BF16, workspace.data(), bytes - 8, &result, nullptr) < 0);
    for (int form = 0; form < 4; ++form) {
      const int bits = form % 2 ? 8 : 32;
      seen = Seen();
      odc_adamw_numbers a = {1e-3, 0.9, 0.999, 1e-8, 0.1, 1.0, 0.0, nullptr, 3, 7, 0, ODC_OPS_F32, ODC_OPS_BF16, ODC_OPS_NONE, bits};
      a.copy_dtype = form < 2 ? ODC_OPS_NONE : ODC_OPS_BF16;
      for (odc_adamw_item& item : items) item.copy = form < 2 ? nullptr : at(0x7000);
      CHECK(odc_adamw(items.data(), (uint32_t)items.size(), &a, nullptr) == ODC_OPS_OK);
      check_tables(seen.adamw, items, adamw_shape(bits == 8).tile());
      uint32_t first = 0;
      for (const AdamwLaunch& launch : seen.adamw) {
        while (first < launch.first_item) CHECK(items[first++].elems == 0);
        CHECK(launch.first_item == first);
        first += launch.n_items;
        CHECK(launch.seed == 7 && std::fabs(launch.step_size - 1e-3 / (1 - 0.9 * 0.9 * 0.9)) < 1e-9);
        CHECK(std::fabs(launch.decay - (1 - 1e-4)) < 1e-7 && std::fabs(launch.one_minus_beta2 - 1e-3) < 1e-9);
      }
    }
  }
}

void check_adamw_refusals() {
  odc_adamw_item item = {at(0x1000), at(0x2000), at(0x3000), at(0x4000), at(0x5001), at(0x6001), nullptr, 100};
  odc_adamw_numbers a = {1e-3, 0.9, 0.999, 1e-8, 0.1, 1.0, 0.0, nullptr, 1, 7, 0, ODC_OPS_F32, ODC_OPS_F32, ODC_OPS_NONE, 32};
  seen = Seen();
  CHECK(odc_adamw(&item, 1, &a, nullptr) == ODC_OPS_OK && seen.adamw.size() == 1);
  const auto refused = [&](auto change) {
    odc_adamw_item it = item;
    odc_adamw_numbers n = a;
    change(it, n);
    CHECK(odc_adamw(&it, 1, &n, nullptr) < 0 && seen.adamw.size() == 1);
  };
  CHECK(odc_adamw(&item, 1, nullptr, nullptr) < 0 && odc_adamw(nullptr, 1, &a, nullptr) < 0);
  refused([](auto& it, auto&) { it.param = nullptr; });
  refused([](auto& it, auto&) { it.grad = nullptr; });
  refused([](auto& it, auto&) { it.exp_avg = at(0x3002); });
  refused([](auto& it, auto&) { it.param = at(0x1002); });
  refused([](auto& it, auto&) { it.copy = at(0x7000); });
  refused([](auto& it, auto& n) { it.copy = at(0x7000), n.copy_dtype = ODC_OPS_F32; });
  refused([](auto& it, auto& n) { it.copy = at(0x7001), n.copy_dtype = ODC_OPS_BF16; });
  refused([](auto&, auto& n) { n.copy_dtype = ODC_OPS_BF16; });
  refused([](auto& it, auto& n) { it.exp_avg_scale = nullptr, n.state_bits = 8; });
  refused([](auto& it, auto&) { it.elems = uint64_t(1) << 50; });
  refused([](auto&, auto& n) { n.state_bits = 16; });
  refused([](auto&, auto& n) { n.param_dtype = ODC_OPS_F16; });
  refused([](auto&, auto& n) { n.grad_dtype = 5; });
  refused([](auto&, auto& n) { n.step = 0; });
  refused([](auto&, auto& n) { n.beta1 = 1; });
  refused([](auto&, auto& n) { n.beta2 = NAN; });
  refused([](auto&, auto& n) { n.lr = -1; });
  refused([](auto&, auto& n) { n.eps = INFINITY; });
  refused([](auto&, auto& n) { n.grad_scale = NAN; });
  refused([](auto&, auto& n) { n.squared_norm = reinterpret_cast<const float*>(at(0x1000)), n.max_norm = NAN; });
  refused([](auto&, auto& n) { n.squared_norm = reinterpret_cast<const float*>(at(0x1002)); });
  answer = 100;
  CHECK(odc_adamw(&item, 1, &a, nullptr) == ODC_OPS_ERR_HIP);
  answer = 0;
  CHECK(odc_dequantize_blocks(at(1), at(2), at(4), 10, ODC_OPS_F32, nullptr) == ODC_OPS_OK && seen.dequantize == 1);
  CHECK(odc_dequantize_blocks(nullptr, at(2), at(4), 10, ODC_OPS_F32, nullptr) < 0);
  CHECK(odc_dequantize_blocks(at(1), at(2), at(2), 10, ODC_OPS_F32, nullptr) < 0);
  CHECK(odc_dequantize_blocks(at(1), at(2), at(4), 10, 7, nullptr) < 0);
  CHECK(odc_dequantize_blocks(nullptr, nullptr, nullptr, 0, ODC_OPS_F32, nullptr) == ODC_OPS_OK && seen.dequantize == 1);
  float result;
  const odc_span_item span = {at(0x1001), 10}, far = {at(uintptr_t(1) << 48), 10};
  CHECK(odc_squared_norm(&far, 1, ODC_OPS_F32, at(0x1000), 1 << 20, &result, nullptr) < 0);
  CHECK(odc_squared_norm(&span, 1, ODC_OPS_F32, at(0x1000), 1 << 20, &result, nullptr) < 0);
  CHECK(odc_squared_norm(&span, 1, 9, at(0x1000), 1 << 20, &result, nullptr) < 0);
  CHECK(odc_squared_norm(&span, 1, ODC_OPS_F32, at(0x1000), 1 << 20, nullptr, nullptr) < 0);
}

}  // namespace

int main() {
  check_layer_norm();
  check_lists();
  check_adamw_refusals();
  puts("ok");
}
