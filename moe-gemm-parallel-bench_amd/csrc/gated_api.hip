// C ABI of the Gate+Up training form: argument checks, the choice of a tile, the launches: one a product (and one for
// dP), another for every further 768 groups or 192 rounds of tiles.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/moegemm.h"
#include "error.h"
#include "gated_train.h"

using namespace moegemm;

namespace {

constexpr int64_t kTwoGiB = int64_t(1) << 31;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// A row pitch in elements: 16-byte rows that cover `width`, 256 of them under 2 GiB.
bool pitch_ok(int64_t pitch, int64_t width) { return pitch % 8 == 0 && pitch >= width && 256 * pitch * 2 < kTwoGiB; }

int check_shape(int32_t group_count, int32_t rows, int32_t h, int32_t f, const int32_t* offs, int32_t dtype) {
  if (dtype != DT_F16 && dtype != DT_BF16)
    return report(MOEGEMM_ERR_INVALID, "the Gate+Up training form needs fp16 or bf16 operands (dtype code %d)", dtype);
  if (group_count <= 0) return report(MOEGEMM_ERR_INVALID, "group_count must be positive (got %d)", group_count);
  if (!offs && group_count != 1)
    return report(MOEGEMM_ERR_INVALID, "without offsets there is one group (got %d)", group_count);
  if (rows < 0 || rows >= 1 << 30 || h <= 0 || f <= 0 || f > 1 << 29)
    return report(MOEGEMM_ERR_INVALID, "bad shape (rows=%d h=%d f=%d)", rows, h, f);
  if (h % 8 || f % 8) return report(MOEGEMM_ERR_INVALID, "h and f must be multiples of 8 (h=%d f=%d)", h, f);
  return MOEGEMM_OK;
}

int check_operand(const char* name, const void* base, int64_t pitch, int64_t width) {
  if (!base) return report(MOEGEMM_ERR_INVALID, "%s must be non-null", name);
  if (!aligned16(base) || !pitch_ok(pitch, width))
    return report(MOEGEMM_ERR_INVALID, "%s rows must start at multiples of 16 bytes and cover %lld elements", name,
                  (long long)width);
  return MOEGEMM_OK;
}

// Row tiles of forward and dX: exact for one group, else about half a tile a group more than the rows fill.
int64_t row_tiles(const GatedVariant& v, int64_t rows, int64_t groups) {
  const int64_t active = std::min(groups, rows);
  return active == 1 ? cdiv(rows, v.block_m) : std::max(active, rows / v.block_m + active / 2);
}

// The variant of the least estimated time: rounds of tiles over the CUs, but no less than reading the weights
// (dW: writing their gradients) takes.  The rounds decide more than a tile's rate does.  16 experts, 4001 rows, 2880 ->
// 2x2880: dX 282 us in two rounds of 256x256 tiles, 187 in two of 128x256; forward 231 against 206.  32 experts, 16384
// rows, 7168 -> 2x2048: forward 977 against 1086.  64 experts of 32 rows, 2048 -> 2x768, bound by the weights: forward
// 102, 92 (128x256), 95, 121 (16x128).  One row, 4096 -> 2x4096: 70, 52, 28, 25.
const GatedVariant* choose(const GatedVariant* list, int product, const GatedParams& p, int64_t cols, int cus) {
  const int64_t k = product == GATED_FORWARD ? p.h : product == GATED_DX ? 2 * (int64_t)p.f : cdiv(p.rows, p.groups);
  const double weights = 4.0 * std::min(p.groups, p.rows) * p.h * p.f;  // bytes
  const GatedVariant* best = nullptr;
  double least = 0;
  for (const GatedVariant* v = list; v->launch; ++v) {
    const int64_t rows = product == GATED_DW ? p.groups * cdiv(p.h, v->block_m) : row_tiles(*v, p.rows, p.groups);
    const int64_t tiles = rows * cdiv(cols, v->block_n), full = tiles / (cus * v->per_cu), rest = tiles % (cus * v->per_cu);
    // A last round that leaves every CU one workgroup takes a round's time by the number a CU holds.
    const double rounds = full + (rest == 0 ? 0.0 : rest <= cus ? 1.0 / v->per_cu : 1.0);
    const double ns = std::max(rounds * k * v->slice_ps * 1e-3 + (full + (rest > 0)) * v->tile_ns, weights / v->gbps);
    if (!best || ns < least) {
      best = v;
      least = ns;
    }
  }
  return best;
}

const GatedTable& table_of(int32_t dtype) { return dtype == DT_BF16 ? kGatedBf16 : kGatedF16; }

// A product's variant, its workgroups and a bound on its tiles.
struct Plan {
  const GatedVariant* v;
  int64_t tiles;
  int grid;
};

int plan_product(const GatedParams& p, int product, int32_t dtype, int32_t variant, int cus, Plan& plan) {
  const GatedVariant* list = table_of(dtype).products[product];
  const int64_t cols = product == GATED_DX ? p.h : 2 * (int64_t)p.f;
  plan.v = nullptr;
  if (variant < 0) {
    plan.v = choose(list, product, p, cols, cus);
  } else {
    for (int i = 0; list[i].launch; ++i)
      if (i == variant) plan.v = &list[i];
    if (!plan.v) return report(MOEGEMM_ERR_NO_KERNEL, "Gate+Up variant %d is not compiled", variant);
  }
  const int bm = plan.v->block_m;
  const int64_t row_tiles = product == GATED_DW
                                ? p.groups * cdiv(p.h, bm)
                                : std::min(p.rows / bm + (int64_t)p.groups, p.groups * cdiv(p.rows, bm));
  plan.tiles = std::max<int64_t>(row_tiles * cdiv(cols, plan.v->block_n), 1);
  if (plan.tiles > INT32_MAX / 2) return report(MOEGEMM_ERR_INVALID, "tile count exceeds int32");
  plan.grid = (int)std::min<int64_t>(plan.tiles, (int64_t)cus * plan.v->per_cu);
  return MOEGEMM_OK;
}

int checked(hipError_t err) {
  return err == hipSuccess ? MOEGEMM_OK
                           : report(MOEGEMM_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(err));
}

int launch_planned(const GatedParams& p, const Plan& plan, hipStream_t stream) {
  GatedParams part = p;
  for (; part.first < p.groups; part.first += kTableGroups) {
    part.groups = std::min(p.groups - part.first, kTableGroups);
    for (part.round = 0; (int64_t)part.round * plan.grid < plan.tiles; part.round += kListTiles) {
      part.closes = part.first + part.groups == p.groups && part.round == 0;
      const int rc = checked(plan.v->launch(part, plan.grid, stream));
      if (rc != MOEGEMM_OK) return rc;
    }
  }
  return MOEGEMM_OK;
}

}  // namespace

extern "C" {

int moegemm_gate_up_variant_count(int32_t product) {
  if (product < 0 || product > 2) return report(MOEGEMM_ERR_INVALID, "product must be 0, 1 or 2 (got %d)", product);
  int count = 0;
  while (kGatedBf16.products[product][count].launch) ++count;
  return count;
}

int moegemm_gate_up_forward(const void* x, const void* w, void* h_out, float* saved, const int32_t* offs,
                            int32_t group_count, int32_t rows, int32_t h, int32_t f, int64_t stride_xm,
                            int64_t stride_wg, int64_t stride_wh, int64_t stride_om, int32_t dtype, int32_t variant,
                            int32_t grid_size, void* stream) {
  int rc = check_shape(group_count, rows, h, f, offs, dtype);
  if (rc == MOEGEMM_OK && rows == 0) return MOEGEMM_OK;
  if (rc == MOEGEMM_OK) rc = check_operand("x", x, stride_xm, h);
  if (rc == MOEGEMM_OK) rc = check_operand("w", w, stride_wh, 2 * (int64_t)f);
  if (rc == MOEGEMM_OK) rc = check_operand("h", h_out, stride_om, f);
  if (rc == MOEGEMM_OK && saved) rc = check_operand("saved", saved, 2 * (int64_t)f, 2 * (int64_t)f);
  if (rc != MOEGEMM_OK) return rc;
  if (stride_wg % 8 || (h + 1024) * stride_wh * 2 >= kTwoGiB)
    return report(MOEGEMM_ERR_INVALID, "a group's weight must start at a multiple of 16 bytes and span under 2 GiB");
  GatedParams p{x, w, h_out, saved, nullptr, offs, stride_xm, stride_wg, stride_wh, stride_om, 0, 0,
                group_count, rows, h, f, 0};
  Plan plan;
  rc = plan_product(p, GATED_FORWARD, dtype, variant, grid_size > 0 ? grid_size : 256, plan);
  return rc == MOEGEMM_OK ? launch_planned(p, plan, reinterpret_cast<hipStream_t>(stream)) : rc;
}

int moegemm_gate_up_backward(const void* dh, const void* x, const void* w, const float* saved, void* dp, void* dx,
                             void* dw, const int32_t* offs, int32_t group_count, int32_t rows, int32_t h, int32_t f,
                             int64_t stride_dhm, int64_t stride_xm, int64_t stride_wg, int64_t stride_wh, int32_t dtype,
                             int32_t dx_variant, int32_t dw_variant, int32_t grid_size, void* stream) {
  const int64_t width = 2 * (int64_t)f;
  int rc = check_shape(group_count, rows, h, f, offs, dtype);
  if (rows > 0) {
    if (rc == MOEGEMM_OK) rc = check_operand("dh", dh, stride_dhm, f);
    if (rc == MOEGEMM_OK) rc = check_operand("saved", saved, width, width);
    if (rc == MOEGEMM_OK) rc = check_operand("dp", dp, width, width);
    if (rc == MOEGEMM_OK && dx) rc = check_operand("w", w, stride_wh, width);
    if (rc == MOEGEMM_OK && dx) rc = check_operand("dx", dx, h, h);
    if (rc == MOEGEMM_OK && dw) rc = check_operand("x", x, stride_xm, h);
  }
  if (rc == MOEGEMM_OK && dw) rc = check_operand("dw", dw, width, width);
  if (rc == MOEGEMM_OK && stride_wg % 8)
    rc = report(MOEGEMM_ERR_INVALID, "a group's weight must start at a multiple of 16 bytes");
  if (rc != MOEGEMM_OK) return rc;
  const hipStream_t queue = reinterpret_cast<hipStream_t>(stream);
  const int cus = grid_size > 0 ? grid_size : 256;
  const GatedTable& table = table_of(dtype);
  const GatedParams of_x{dp, w, dx, nullptr, nullptr, offs, width, stride_wg, stride_wh, h, 0, 0,
                         group_count, rows, h, f, 0};
  const GatedParams of_w{x, nullptr, dw, nullptr, dp, offs, stride_xm, 0, 0, width, h * width, width,
                         group_count, rows, h, f,
                         (rows + (int64_t)1024) * std::max<int64_t>(stride_xm, width) * 2 >= kTwoGiB};
  const bool want_dx = dx && rows > 0;
  Plan plan_x{}, plan_w{};
  if (want_dx) rc = plan_product(of_x, GATED_DX, dtype, dx_variant, cus, plan_x);
  if (rc == MOEGEMM_OK && dw) rc = plan_product(of_w, GATED_DW, dtype, dw_variant, cus, plan_w);
  if (rc != MOEGEMM_OK) return rc;

  if (rows > 0 && (dx || dw)) {
    const GatedParams p{nullptr, nullptr, nullptr, const_cast<float*>(saved), nullptr, offs, 0, 0, 0, 0, 0, 0,
                        group_count, rows, h, f, 0};
    const int64_t blocks = cdiv((int64_t)rows * (f / 8), 256);
    rc = checked(table.gradient(p, dh, stride_dhm, dp, (int)std::min<int64_t>(blocks, cus * 16), queue));
    if (rc != MOEGEMM_OK) return rc;
  }
  if (want_dx) rc = launch_planned(of_x, plan_x, queue);
  if (rc == MOEGEMM_OK && dw) rc = launch_planned(of_w, plan_w, queue);
  return rc;
}

}  // extern "C"
