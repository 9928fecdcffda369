// C ABI of the routing operators: argument checks and launches.  One launch a call; a sort of more than one chunk is
// two.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/moegemm.h"
#include "error.h"
#include "routing.h"

using namespace moegemm;

namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int checked(hipError_t err) {
  return err == hipSuccess ? MOEGEMM_OK
                           : report(MOEGEMM_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(err));
}

int64_t element_bytes(int32_t dtype) { return dtype == DT_F32 ? 4 : 2; }

int check_route(const RouteParams& p, int32_t dtype) {
  if (dtype != DT_F16 && dtype != DT_BF16 && dtype != DT_F32)
    return report(MOEGEMM_ERR_INVALID, "unsupported dtype code %d", dtype);
  if (p.tokens < 0 || p.experts <= 0 || p.experts > kRouteExperts)
    return report(MOEGEMM_ERR_INVALID, "bad shape (tokens=%d experts=%d, at most %d experts)", p.tokens, p.experts,
                  kRouteExperts);
  if (p.k <= 0 || p.k > kRouteTop || p.k > p.experts)
    return report(MOEGEMM_ERR_INVALID, "k must be 1 to min(experts, %d) (got %d)", kRouteTop, p.k);
  if ((p.sigmoid != 0 && p.sigmoid != 1) || (p.normalize != 0 && p.normalize != 1))
    return report(MOEGEMM_ERR_INVALID, "sigmoid and normalize must be 0 or 1");
  if (!p.logits && p.tokens) return report(MOEGEMM_ERR_INVALID, "logits must be non-null");
  if (!aligned(p.logits, element_bytes(dtype)))
    return report(MOEGEMM_ERR_INVALID, "logits must be aligned to their element size");
  return MOEGEMM_OK;
}

constexpr int64_t kMaxBlocks = 1 << 16;  // workgroups of a launch; they go on to the tokens and rows past them

// Whether route_kernel can choose: k on a list of `top` with two to spare where scores may be too close to call, and
// groups that are whole lanes' experts, as many to each.  Else every token takes the 64-bit path (16384 tokens, 8 of
// 256 experts, sigmoid with a bias: 11.2 us and 43.9; 4 of 8 groups 15.2 and 63.8).
template <class E, RouteRank RANK>
bool fast_route(const RouteParams& p, int lanes, int top) {
  return p.k <= (RANK >= RANK_SIGMOID || E::is_f32 ? top - 2 : top) &&
         (p.groups == 1 || (p.groups <= 16 && lanes % p.groups == 0 && p.experts % lanes == 0));
}

dim3 route_grid(const RouteParams& p, int64_t tokens) { return dim3((unsigned)cdiv(p.tokens, tokens)); }
size_t route_lds(const RouteParams& p) { return 4 * (p.experts + p.groups) * sizeof(uint64_t); }  // at most 64 KiB

template <class E, int LPT, int PER, int TOP, RouteRank RANK>
hipError_t launch_choice(const RouteParams& p, hipStream_t stream) {
  hipLaunchKernelGGL((route_kernel<E, LPT, PER, TOP, RANK>), route_grid(p, 256 / LPT), dim3(256), route_lds(p), stream, p);
  return hipGetLastError();
}
// 16 lanes a token for lists of 16 from up to 256 experts, else all 64 (16384 tokens, 256 experts by fp32 logits: 14 by 16
// lanes and a list of 16 9.4 us, 15 by 64 lanes and a list of 32 44).  A list of 32 against the 64-bit path, which it
// stands in front of for 15 to 30 (WHOLE: 17 to 32) experts: 15 of 256 44 and 70 us, 30 of 256 45 and 127; 4097 tokens, 15
// of 896 20 and 53, 30 of 896 19 and 93; 64 tokens, 15 of 256 5.0 and 19.7.
template <class E, RouteRank RANK>
hipError_t launch_choice(const RouteParams& p, hipStream_t stream) {
  if (p.experts <= 256 && fast_route<E, RANK>(p, 16, 16)) {
    const int64_t per = cdiv(p.experts, 16);
    return per <= 4   ? launch_choice<E, 16, 4, 16, RANK>(p, stream)
           : per <= 8 ? launch_choice<E, 16, 8, 16, RANK>(p, stream)
                      : launch_choice<E, 16, 16, 16, RANK>(p, stream);
  }
  if (p.experts > 256 && fast_route<E, RANK>(p, 64, 16))
    return p.experts <= 512 ? launch_choice<E, 64, 8, 16, RANK>(p, stream) : launch_choice<E, 64, 16, 16, RANK>(p, stream);
  if (fast_route<E, RANK>(p, 64, 32))
    return p.experts <= 256 ? launch_choice<E, 64, 4, 32, RANK>(p, stream) : launch_choice<E, 64, 16, 32, RANK>(p, stream);
  hipLaunchKernelGGL((route_exact_kernel<E>), route_grid(p, 4), dim3(256), route_lds(p), stream, p);
  return hipGetLastError();
}
template <class E, int LPT, int PER>
hipError_t launch_gradient(const RouteParams& p, hipStream_t stream) {
  hipLaunchKernelGGL((route_backward_kernel<E, LPT, PER>), route_grid(p, 256 / LPT), dim3(256), 0, stream, p);
  return hipGetLastError();
}
// 16 lanes a token up to 16 chosen of 256 experts, else all 64 (16384 tokens, 256 experts: 16 chosen by 16 lanes 6.4 us, 17 by
// 64 lanes 8.6; dense 10.6 and 12.4).
template <class E>
hipError_t launch_gradient(const RouteParams& p, hipStream_t stream) {
  if (p.k <= 16 && p.experts <= 256) {
    const int64_t per = cdiv(p.experts, 16);
    return per <= 4   ? launch_gradient<E, 16, 4>(p, stream)
           : per <= 8 ? launch_gradient<E, 16, 8>(p, stream)
                      : launch_gradient<E, 16, 16>(p, stream);
  }
  return p.experts <= 256   ? launch_gradient<E, 64, 4>(p, stream)
         : p.experts <= 512 ? launch_gradient<E, 64, 8>(p, stream)
                            : launch_gradient<E, 64, 16>(p, stream);
}
template <class E>
hipError_t launch_route(const RouteParams& p, bool backward, hipStream_t stream) {
  if (backward) return launch_gradient<E>(p, stream);
  if (p.bias || p.group_best == 2)
    return p.sigmoid ? launch_choice<E, RANK_SIGMOID>(p, stream) : launch_choice<E, RANK_SOFTMAX>(p, stream);
  return p.sigmoid || p.normalize ? launch_choice<E, RANK_LOGITS>(p, stream) : launch_choice<E, RANK_LOGITS_SUM>(p, stream);
}
int launch_route(RouteParams p, bool backward, int32_t dtype, void* stream) {
  constexpr int32_t kTokens = 1 << 25;  // of a launch: it counts threads in 32 bits, at most 64 a token
  const auto s = reinterpret_cast<hipStream_t>(stream);
  const int64_t es = element_bytes(dtype);
  for (int32_t left = p.tokens; left > 0; left -= kTokens) {
    p.tokens = std::min(left, kTokens);
    const int rc = checked(dtype == DT_F32    ? launch_route<EF32>(p, backward, s)
                           : dtype == DT_BF16 ? launch_route<EBf16>(p, backward, s)
                                              : launch_route<EF16>(p, backward, s));
    if (rc != MOEGEMM_OK) return rc;
    const int64_t picks = (int64_t)p.tokens * p.k;
    p.logits = static_cast<const char*>(p.logits) + p.tokens * p.ldl * es;
    p.chosen += picks;
    if (backward) {
      p.dweights += picks;
      p.dlogits = static_cast<char*>(p.dlogits) + (int64_t)p.tokens * p.experts * es;
    } else {
      p.weights += picks;
    }
  }
  return MOEGEMM_OK;
}

// Up to so many entries one workgroup sorts all of them (us, one launch and two: 512 entries 4.0 and 8.4, 4096 6.4 and
// 8.9, 8192 9.9 and 9.1, but the second launch takes the host 3 us more).
constexpr int64_t kSortWhole = 8192;
// Entries of a workgroup of the others: 64 workgroups, or more of 16384 entries up to 256, since each reads all counts.
int64_t sort_chunk(int64_t n) {
  return cdiv(std::max({std::min(cdiv(n, 64), int64_t(16384)), cdiv(n, 256), int64_t(1024)}), 1024) * 1024;
}

// The widest unit that rows and their pitches allow.
int64_t unit_bytes(int64_t width, std::initializer_list<std::pair<const void*, int64_t>> rows) {
  int64_t unit = 16;
  auto fits = [&](int64_t u) {
    if (width % u) return false;
    for (const auto& r : rows)
      if (r.first && (!aligned(r.first, u) || r.second % u)) return false;
    return true;
  };
  while (unit > 1 && !fits(unit)) unit >>= 1;
  return unit;
}

using U16 = u32x4_t;

// `end` may be null where no rows are cleared.
int check_rows(int64_t tokens, int32_t k, int32_t rows, int64_t width, const int32_t* places, const int32_t* end, bool clears) {
  if (tokens < 0 || tokens > INT32_MAX || k <= 0 || rows < 0 || width <= 0 || width > INT32_MAX)
    return report(MOEGEMM_ERR_INVALID, "bad shape (tokens=%lld k=%d rows=%d, rows of %lld bytes)", (long long)tokens, k,
                  rows, (long long)width);
  if ((!places && tokens) || (!end && clears)) return report(MOEGEMM_ERR_INVALID, "places and offs must be non-null");
  return MOEGEMM_OK;
}

// Whether the sorted rows go past the caches: from 128 MiB of them on (8 rows a token of 14336 bytes, us for combine,
// its gradients and gather: 59 MB kept 11.8, 18.9, 10.1, past 12.3, 28.1, 11.9; 117 MB 25.5, 47.0, 24.0 and 23.6, 48.4,
// 23.8; 470 MB 106, 207, 106 and 92, 194, 95).
bool past_caches(int64_t rows, int64_t width, int64_t unit) { return unit == 16 && rows * width >= int64_t(128) << 20; }

template <class E>
hipError_t launch_combine(const RowsParams& p, int64_t unit, dim3 grid, hipStream_t s) {
  using raw = typename E::raw;
  if (past_caches(p.rows, p.width, unit)) hipLaunchKernelGGL((combine_rows_kernel<E, U16, true>), grid, dim3(256), 0, s, p);
  else if (unit == 16) hipLaunchKernelGGL((combine_rows_kernel<E, U16, false>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((combine_rows_kernel<E, raw, false>), grid, dim3(256), 0, s, p);
  return hipGetLastError();
}
template <class E>
hipError_t launch_combine_backward(const RowsParams& p, int64_t unit, dim3 grid, hipStream_t s) {
  using raw = typename E::raw;
  if (past_caches(p.rows, p.width, unit))
    hipLaunchKernelGGL((combine_rows_backward_kernel<E, U16, true>), grid, dim3(256), 0, s, p);
  else if (unit == 16) hipLaunchKernelGGL((combine_rows_backward_kernel<E, U16, false>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((combine_rows_backward_kernel<E, raw, false>), grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace

extern "C" {

int moegemm_route_topk(const void* logits, const float* bias, float* weights, int32_t* experts, int32_t tokens,
                       int32_t expert_count, int32_t k, int64_t stride_lt, int32_t dtype, int32_t sigmoid, int32_t groups,
                       int32_t top_groups, int32_t group_best, int32_t normalize, float scale, void* stream) {
  RouteParams p{logits, bias, weights, experts, nullptr, nullptr, stride_lt, tokens, expert_count, k, sigmoid, groups,
                top_groups, group_best, normalize, scale};
  const int rc = check_route(p, dtype);
  if (rc != MOEGEMM_OK) return rc;
  if (groups <= 0 || expert_count % groups || top_groups <= 0 || top_groups > groups || (group_best != 1 && group_best != 2))
    return report(MOEGEMM_ERR_INVALID, "bad expert groups (%d of %d over %d experts, group_best %d)", top_groups, groups,
                  expert_count, group_best);
  if (k > top_groups * (expert_count / groups))
    return report(MOEGEMM_ERR_INVALID, "k = %d experts do not fit %d groups of %d", k, top_groups, expert_count / groups);
  if (tokens == 0) return MOEGEMM_OK;
  if (!weights || !experts) return report(MOEGEMM_ERR_INVALID, "weights and experts must be non-null");
  return launch_route(p, false, dtype, stream);
}

int moegemm_route_topk_backward(const float* dweights, const void* logits, const int32_t* experts, void* dlogits,
                                int32_t tokens, int32_t expert_count, int32_t k, int64_t stride_lt, int32_t dtype,
                                int32_t sigmoid, int32_t normalize, float scale, void* stream) {
  RouteParams p{logits, nullptr, nullptr, const_cast<int32_t*>(experts), dweights, dlogits, stride_lt, tokens, expert_count,
                k, sigmoid, 1, 1, 1, normalize, scale};
  const int rc = check_route(p, dtype);
  if (rc != MOEGEMM_OK || tokens == 0) return rc;
  if (!dweights || !experts || !dlogits) return report(MOEGEMM_ERR_INVALID, "dweights, experts and dlogits must be non-null");
  if (!aligned(dlogits, element_bytes(dtype)))
    return report(MOEGEMM_ERR_INVALID, "dlogits must be aligned to its element size");
  return launch_route(p, true, dtype, stream);
}

int64_t moegemm_sort_workspace_bytes(int64_t entries, int32_t count) {
  if (entries < 0 || entries > INT32_MAX || count <= 0 || count > kSortExperts)
    return report(MOEGEMM_ERR_INVALID, "bad sort (%lld entries, %d experts of at most %d)", (long long)entries, count,
                  kSortExperts);
  return entries <= kSortWhole ? 0 : cdiv(entries, sort_chunk(entries)) * count * 4;
}

int moegemm_sort_by_expert(const int32_t* experts, int32_t* offs, int32_t* slots, int32_t* places, int32_t entries,
                           int32_t first, int32_t count, void* workspace, int64_t workspace_bytes, void* stream) {
  const int64_t need = moegemm_sort_workspace_bytes(entries, count);
  if (need < 0) return (int)need;
  if (first < 0) return report(MOEGEMM_ERR_INVALID, "the first expert must not be negative (got %d)", first);
  if (!offs || (!workspace && need) || (entries && (!experts || !slots || !places)))
    return report(MOEGEMM_ERR_INVALID, "experts, offs, slots, places and workspace must be non-null");
  if (workspace_bytes < need)
    return report(MOEGEMM_ERR_INVALID, "the workspace holds %lld bytes of %lld", (long long)workspace_bytes, (long long)need);
  const auto s = reinterpret_cast<hipStream_t>(stream);
  const bool whole = entries <= kSortWhole;
  const int64_t chunk = sort_chunk(entries);
  SortParams p{experts, offs, slots, places, static_cast<int32_t*>(workspace), entries, first, count, (int32_t)chunk};
  if (whole) {
    const size_t lds = 16 * count * sizeof(int32_t);
    if (entries <= 1024) hipLaunchKernelGGL(sort_whole_kernel<1>, dim3(1), dim3(1024), lds, s, p);
    else if (entries <= 4096) hipLaunchKernelGGL(sort_whole_kernel<4>, dim3(1), dim3(1024), lds, s, p);
    else hipLaunchKernelGGL(sort_whole_kernel<8>, dim3(1), dim3(1024), lds, s, p);
    return checked(hipGetLastError());
  }
  const dim3 grid((unsigned)cdiv(entries, chunk));
  hipLaunchKernelGGL(sort_count_kernel, grid, dim3(256), 0, s, p);
  const int rc = checked(hipGetLastError());
  if (rc != MOEGEMM_OK) return rc;
  hipLaunchKernelGGL(sort_place_kernel, grid, dim3(256), 0, s, p);
  return checked(hipGetLastError());
}

int moegemm_gather_rows(const void* x, void* out, const int32_t* places, const int32_t* end, int64_t tokens, int32_t k,
                        int32_t rows, int64_t row_bytes, int64_t stride_x, int64_t stride_out, void* stream) {
  const int rc = check_rows(tokens, k, rows, row_bytes, places, end, true);
  if (rc != MOEGEMM_OK || rows == 0) return rc;
  if ((!x && tokens) || !out) return report(MOEGEMM_ERR_INVALID, "x and out must be non-null");
  const int64_t unit = unit_bytes(row_bytes, {{x, stride_x}, {out, stride_out}});
  const int64_t spans = cdiv(row_bytes, 4 * 64 * unit);
  const RowsParams p{static_cast<const char*>(x), static_cast<char*>(out), places, end, nullptr, nullptr, nullptr, stride_x,
                     stride_out, 0, tokens, k, rows, (int32_t)row_bytes, (int32_t)spans};
  const dim3 grid((unsigned)(kClearBlocks + std::min(cdiv(tokens * spans, 4), kMaxBlocks)));
  const auto s = reinterpret_cast<hipStream_t>(stream);
  switch (unit) {
    case 16:
      if (past_caches(rows, row_bytes, unit)) hipLaunchKernelGGL((gather_rows_kernel<U16, true>), grid, dim3(256), 0, s, p);
      else hipLaunchKernelGGL((gather_rows_kernel<U16, false>), grid, dim3(256), 0, s, p);
      break;
    case 8: hipLaunchKernelGGL((gather_rows_kernel<uint64_t, false>), grid, dim3(256), 0, s, p); break;
    case 4: hipLaunchKernelGGL((gather_rows_kernel<uint32_t, false>), grid, dim3(256), 0, s, p); break;
    case 2: hipLaunchKernelGGL((gather_rows_kernel<uint16_t, false>), grid, dim3(256), 0, s, p); break;
    default: hipLaunchKernelGGL((gather_rows_kernel<uint8_t, false>), grid, dim3(256), 0, s, p);
  }
  return checked(hipGetLastError());
}

int moegemm_combine_rows(const void* y, const float* weights, void* out, const int32_t* places, int64_t tokens, int32_t k,
                         int32_t rows, int32_t width, int64_t stride_y, int64_t stride_out, int32_t dtype, void* stream) {
  if (dtype != DT_F16 && dtype != DT_BF16 && dtype != DT_F32)
    return report(MOEGEMM_ERR_INVALID, "unsupported dtype code %d", dtype);
  const int64_t es = element_bytes(dtype);
  const int rc = check_rows(tokens, k, rows, width * es, places, nullptr, false);
  if (rc != MOEGEMM_OK || tokens == 0) return rc;
  if ((!y && rows) || !out) return report(MOEGEMM_ERR_INVALID, "y and out must be non-null");
  if (!aligned(y, es) || !aligned(out, es))
    return report(MOEGEMM_ERR_INVALID, "y and out must be aligned to their element size");
  const int64_t unit = unit_bytes(width * es, {{y, stride_y * es}, {out, stride_out * es}}) == 16 ? 16 : es;
  const int64_t spans = cdiv(width * es, 2 * 64 * unit);
  const RowsParams p{static_cast<const char*>(y), static_cast<char*>(out), places, nullptr, weights, nullptr, nullptr,
                     stride_y * es, stride_out * es, 0, tokens, k, rows, (int32_t)(width * es), (int32_t)spans};
  const dim3 grid((unsigned)std::min(cdiv(tokens * spans, 4), kMaxBlocks));
  const auto s = reinterpret_cast<hipStream_t>(stream);
  return checked(dtype == DT_F32    ? launch_combine<EF32>(p, unit, grid, s)
                 : dtype == DT_BF16 ? launch_combine<EBf16>(p, unit, grid, s)
                                    : launch_combine<EF16>(p, unit, grid, s));
}

int moegemm_combine_rows_backward(const void* dout, const void* y, const float* weights, void* dy, float* dweights,
                                  const int32_t* places, const int32_t* end, int64_t tokens, int32_t k, int32_t rows,
                                  int32_t width, int64_t stride_dout, int64_t stride_y, int32_t dtype, void* stream) {
  if (dtype != DT_F16 && dtype != DT_BF16 && dtype != DT_F32)
    return report(MOEGEMM_ERR_INVALID, "unsupported dtype code %d", dtype);
  const int64_t es = element_bytes(dtype);
  const int rc = check_rows(tokens, k, rows, width * es, places, end, true);
  if (rc != MOEGEMM_OK || (!dy && !dweights)) return rc;
  if ((!dout && tokens) || (dweights && rows && !y))
    return report(MOEGEMM_ERR_INVALID, "dout, and y where dweights is wanted, must be non-null");
  if (!aligned(y, es) || !aligned(dout, es) || !aligned(dy, es))
    return report(MOEGEMM_ERR_INVALID, "dout, y and dy must be aligned to their element size");
  const int64_t unit =
      unit_bytes(width * es, {{dweights ? y : nullptr, stride_y * es}, {dout, stride_dout * es}, {dy, 0}}) == 16 ? 16 : es;
  const RowsParams p{static_cast<const char*>(y), static_cast<char*>(dy), places, end, weights, static_cast<const char*>(dout),
                     dweights, stride_y * es, width * es, stride_dout * es, tokens, k, rows, (int32_t)(width * es), 1};
  const dim3 grid((unsigned)(kClearBlocks + std::min(cdiv(tokens * k, 4), kMaxBlocks)));
  const auto s = reinterpret_cast<hipStream_t>(stream);
  return checked(dtype == DT_F32    ? launch_combine_backward<EF32>(p, unit, grid, s)
                 : dtype == DT_BF16 ? launch_combine_backward<EBf16>(p, unit, grid, s)
                                    : launch_combine_backward<EF16>(p, unit, grid, s));
}

}  // extern "C"
