// C ABI of the Gate+Up training form: argument checks, the choice of a tile, one launch each.
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
    const int64_t rounds = cdiv(rows * cdiv(cols, v->block_n), (int64_t)cus * v->per_cu);
    const double ns = std::max(rounds * (k * v->slice_ps * 1e-3 + v->tile_ns), weights / v->gbps);
    if (!best || ns < least) {
      best = v;
      least = ns;
    }
  }
  return best;
}

const GatedTable& table_of(int32_t dtype) { return dtype == DT_BF16 ? kGatedBf16 : kGatedF16; }

int launch_product(const GatedParams& p, int product, int32_t dtype, int32_t variant, int32_t grid_size, void* stream) {
  const GatedVariant* list = table_of(dtype).products[product];
  const int cus = grid_size > 0 ? grid_size : 256;
  const int64_t cols = product == GATED_DX ? p.h : 2 * (int64_t)p.f;
  const GatedVariant* v = nullptr;
  if (variant < 0) {
    v = choose(list, product, p, cols, cus);
  } else {
    for (int i = 0; list[i].launch; ++i)
      if (i == variant) v = &list[i];
    if (!v) return report(MOEGEMM_ERR_NO_KERNEL, "Gate+Up variant %d is not compiled", variant);
  }
  const int64_t row_tiles = product == GATED_DW
                                ? p.groups * cdiv(p.h, v->block_m)
                                : std::min(p.rows / v->block_m + (int64_t)p.groups, p.groups * cdiv(p.rows, v->block_m));
  const int64_t bound = row_tiles * cdiv(cols, v->block_n);
  if (bound > INT32_MAX / 2) return report(MOEGEMM_ERR_INVALID, "tile count exceeds int32");
  const int grid = (int)std::min<int64_t>(std::max<int64_t>(bound, 1), (int64_t)cus * v->per_cu);
  GatedParams part = p;
  for (; part.first < p.groups; part.first += kTableGroups) {
    part.groups = std::min(p.groups - part.first, kTableGroups);
    for (part.round = 0; (int64_t)part.round * grid < std::max<int64_t>(bound, 1); part.round += kListTiles) {
      part.closes = part.first + part.groups == p.groups && part.round == 0;
      const hipError_t err = v->launch(part, grid, reinterpret_cast<hipStream_t>(stream));
      if (err != hipSuccess) return report(MOEGEMM_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(err));
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
  if (rc == MOEGEMM_OK) rc = check_operand("saved", saved, 2 * (int64_t)f, 2 * (int64_t)f);
  if (rc != MOEGEMM_OK) return rc;
  if (stride_wg % 8 || (h + 1024) * stride_wh * 2 >= kTwoGiB)
    return report(MOEGEMM_ERR_INVALID, "a group's weight must start at a multiple of 16 bytes and span under 2 GiB");
  GatedParams p{x, w, h_out, saved, nullptr, offs, stride_xm, stride_wg, stride_wh, stride_om, 0, 0,
                group_count, rows, h, f, 0};
  return launch_product(p, GATED_FORWARD, dtype, variant, grid_size, stream);
}

int moegemm_gate_up_gradient(const void* dh, const float* saved, void* dp, const int32_t* offs, int32_t group_count,
                             int32_t rows, int32_t f, int64_t stride_dhm, int32_t dtype, int32_t grid_size,
                             void* stream) {
  int rc = check_shape(group_count, rows, 8, f, offs, dtype);
  if (rc == MOEGEMM_OK && rows == 0) return MOEGEMM_OK;
  if (rc == MOEGEMM_OK) rc = check_operand("dh", dh, stride_dhm, f);
  if (rc == MOEGEMM_OK) rc = check_operand("saved", saved, 2 * (int64_t)f, 2 * (int64_t)f);
  if (rc == MOEGEMM_OK) rc = check_operand("dp", dp, 2 * (int64_t)f, 2 * (int64_t)f);
  if (rc != MOEGEMM_OK) return rc;
  GatedParams p{nullptr, nullptr, nullptr, const_cast<float*>(saved), nullptr, offs, 0, 0, 0, 0, 0, 0,
                group_count, rows, 8, f, 0};
  const int64_t blocks = cdiv((int64_t)rows * (f / 8), 256), cus = grid_size > 0 ? grid_size : 256;
  const hipError_t err = table_of(dtype).gradient(p, dh, stride_dhm, dp, (int)std::min<int64_t>(blocks, cus * 16),
                                                  reinterpret_cast<hipStream_t>(stream));
  if (err != hipSuccess) return report(MOEGEMM_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(err));
  return MOEGEMM_OK;
}

int moegemm_gate_up_dx(const void* dp, const void* w, void* dx, const int32_t* offs, int32_t group_count, int32_t rows,
                       int32_t h, int32_t f, int64_t stride_wg, int64_t stride_wh, int64_t stride_om, int32_t dtype,
                       int32_t variant, int32_t grid_size, void* stream) {
  int rc = check_shape(group_count, rows, h, f, offs, dtype);
  if (rc == MOEGEMM_OK && rows == 0) return MOEGEMM_OK;
  if (rc == MOEGEMM_OK) rc = check_operand("dp", dp, 2 * (int64_t)f, 2 * (int64_t)f);
  if (rc == MOEGEMM_OK) rc = check_operand("w", w, stride_wh, 2 * (int64_t)f);
  if (rc == MOEGEMM_OK) rc = check_operand("dx", dx, stride_om, h);
  if (rc != MOEGEMM_OK) return rc;
  if (stride_wg % 8) return report(MOEGEMM_ERR_INVALID, "a group's weight must start at a multiple of 16 bytes");
  GatedParams p{dp, w, dx, nullptr, nullptr, offs, 2 * (int64_t)f, stride_wg, stride_wh, stride_om, 0, 0,
                group_count, rows, h, f, 0};
  return launch_product(p, GATED_DX, dtype, variant, grid_size, stream);
}

int moegemm_gate_up_dw(const void* x, const void* dp, void* dw, const int32_t* offs, int32_t group_count, int32_t rows,
                       int32_t h, int32_t f, int64_t stride_xm, int64_t stride_og, int64_t stride_oh, int32_t dtype,
                       int32_t variant, int32_t grid_size, void* stream) {
  int rc = check_shape(group_count, rows, h, f, offs, dtype);
  if (rc == MOEGEMM_OK && rows > 0) rc = check_operand("x", x, stride_xm, h);
  if (rc == MOEGEMM_OK && rows > 0) rc = check_operand("dp", dp, 2 * (int64_t)f, 2 * (int64_t)f);
  if (rc == MOEGEMM_OK) rc = check_operand("dw", dw, stride_oh, 2 * (int64_t)f);
  if (rc != MOEGEMM_OK) return rc;
  if (stride_og % 8) return report(MOEGEMM_ERR_INVALID, "a group's dw must start at a multiple of 16 bytes");
  const int64_t pitch = std::max<int64_t>(stride_xm, 2 * (int64_t)f);
  GatedParams p{x, nullptr, dw, nullptr, dp, offs, stride_xm, 0, 0, stride_oh, stride_og, 2 * (int64_t)f,
                group_count, rows, h, f, (rows + (int64_t)1024) * pitch * 2 >= kTwoGiB};
  return launch_product(p, GATED_DW, dtype, variant, grid_size, stream);
}

}  // extern "C"
