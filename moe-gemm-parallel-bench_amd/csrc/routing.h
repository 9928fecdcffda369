// Routing (gfx950): each token's experts from the router's logits, and the way to expert-sorted rows and back.
//
//   route      s = softmax(x) or sigmoid(x) over a token's E experts; c = s + bias chooses (the bias only chooses):
//              of equal consecutive groups of experts the top_groups ones with the largest sums of their group_best best c
//              are kept, of those the k experts of the largest c; ties go to the lowest index.
//              w = s of the chosen, over their sum if normalised, times scale.
//   sort       a stable counting sort of the T x k chosen experts: offs (end rows), slots (sorted row -> t k + j) and
//              places (slot -> sorted row, -1 for experts that are not this call's).
//   gather     xs[places[t, j]] = x[t];  combine  out[t] = sum_j w[t, j] y[places[t, j]];  and combine's gradients
//              dy[places[t, j]] = w[t, j] dout[t], dw[t, j] = <dout[t], y[places[t, j]]>.
#pragma once

#include "gemm_kernel.h"

namespace moegemm {

constexpr int kRouteExperts = 1024;  // 16 scores a lane
constexpr int kRouteTop = 64;        // one chosen expert a lane
constexpr int kSortExperts = 1024;   // counters of four waves in 16 KiB of LDS

template <class E>
__device__ __forceinline__ float to_float(typename E::raw r) {
  if constexpr (E::dtype == DT_F32) return __builtin_bit_cast(float, r);
  else if constexpr (E::dtype == DT_BF16) return __builtin_bit_cast(float, (uint32_t)r << 16);
  else return (float)__builtin_bit_cast(_Float16, r);
}
template <class E>
__device__ __forceinline__ typename E::raw from_float(float v) {
  if constexpr (E::dtype == DT_F32) return __builtin_bit_cast(uint32_t, v);
  else if constexpr (E::dtype == DT_BF16) return __builtin_bit_cast(uint16_t, (__bf16)v);
  else return __builtin_bit_cast(uint16_t, (_Float16)v);
}

struct RouteParams {
  const void* logits;  // [tokens, experts], ldl elements between rows
  const float* bias;   // [experts] or null
  float* weights;      // [tokens, k]
  int32_t* chosen;     // [tokens, k]
  const float* dweights;
  void* dlogits;       // [tokens, experts], contiguous
  int64_t ldl;
  int32_t tokens, experts, k, sigmoid, groups, top_groups, group_best, normalize;
  float scale;
};

// Scores as integers of the same order; a NaN lies below -inf, and 0 below everything is "not to be had".
__device__ __forceinline__ uint64_t order_of(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return x != x ? 1 : u >> 63 ? ~u : u | (1ull << 63);
}

struct Best {
  uint64_t key;
  int index;
};
__device__ __forceinline__ void better(Best& a, uint64_t key, int index) {
  if (key > a.key || (key == a.key && index < a.index)) a = {key, index};
}
__device__ __forceinline__ Best wave_best(Best b) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t key = __shfl_xor(b.key, d);
    const int index = __shfl_xor(b.index, d);
    better(b, key, index);
  }
  return b;
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
  return x;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}
__device__ __forceinline__ double sigmoid64(double x) { return 1.0 / (1.0 + exp(-x)); }

// max of a softmax: 0 where nothing is above -inf, so that exp(x - max) is 0 there and not NaN.
__device__ __forceinline__ float softmax_base(float top) { return top == -__builtin_inff() ? 0.0f : top; }

// One token a wave.  Selection runs on 64-bit scores, so that which of two close ones is larger never hangs on a
// rounding of exp; PER scores a lane, expert lane + 64 i.
template <class E, int PER>
__device__ __forceinline__ void route_token(const RouteParams& p, int64_t t, int lane, double* s_score) {
  const typename E::raw* x = static_cast<const typename E::raw*>(p.logits) + t * p.ldl;
  float v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = lane + 64 * i < p.experts ? to_float<E>(x[lane + 64 * i]) : -__builtin_inff();
  bool nan = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) nan |= v[i] != v[i];
  nan = __ballot(nan) != 0;
  // Without a bias, and unless scores are added up, they rank as the logits do.
  const bool by_logit = !p.bias && p.group_best == 1;
  double s[PER];
  float base = 0;
  double total = 1;
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = by_logit ? (double)v[i] : sigmoid64(v[i]);
  } else {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) top = fmaxf(top, v[i]);
    base = softmax_base(wave_max(top));
    total = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s[i] = exp((double)v[i] - base);
      total += s[i];
    }
    total = wave_sum(total);
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = by_logit ? (double)v[i] : total == 0 ? 0 : s[i] / total;
  }
  uint64_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 64 * i;
    key[i] = e < p.experts ? order_of(p.bias ? s[i] + p.bias[e] : s[i]) : 0;
  }
  if (p.groups > 1) {
    // A group a lane in turn: its best scores one after the other, then the best groups.
    const int size = p.experts / p.groups;
    auto score_of = [](uint64_t k) {
      return k == 1 ? __builtin_nan("") : __builtin_bit_cast(double, k >> 63 ? k ^ (1ull << 63) : ~k);
    };
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 64 * i < p.experts) s_score[lane + 64 * i] = score_of(key[i]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint64_t kept[PER] = {};  // of groups lane + 64 i
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int g = lane + 64 * i;
      if (g >= p.groups) continue;
      uint64_t first = 0, second = 0;
      for (int e = 0; e < size; ++e) {
        const uint64_t c = order_of(s_score[g * size + e]);
        if (c > first) {
          second = first;
          first = c;
        } else if (c > second) {
          second = c;
        }
      }
      const double sum = p.group_best == 2 && size > 1 ? score_of(first) + score_of(second) : score_of(first);
      kept[i] = order_of(sum);
    }
    uint32_t of_group[PER] = {};
    for (int n = 0; n < p.top_groups; ++n) {
      Best b{0, 0};
#pragma unroll
      for (int i = 0; i < PER; ++i) better(b, kept[i], lane + 64 * i);
      b = wave_best(b);
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (b.index == lane + 64 * i) {
          kept[i] = 0;
          of_group[i] = 1;
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) s_score[lane + 64 * i] = of_group[i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 64 * i < p.experts && s_score[(lane + 64 * i) / size] == 0) key[i] = 0;
  }
  int mine = 0;
  for (int j = 0; j < p.k; ++j) {
    Best b{0, 0};
#pragma unroll
    for (int i = 0; i < PER; ++i) better(b, key[i], lane + 64 * i);
    b = wave_best(b);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (b.index == lane + 64 * i) key[i] = 0;
    if (lane == j) mine = b.index;
  }
  const bool used = lane < p.k;
  const float logit = used ? to_float<E>(x[mine]) : -__builtin_inff();
  double w;
  if (p.sigmoid) {
    w = used ? sigmoid64(logit) : 0;
    if (p.normalize) {
      const double sum = wave_sum(w);
      w = sum == 0 ? 0 : w / sum;
    }
  } else {
    // Normalised: a softmax of the chosen ones alone.
    if (p.normalize) base = softmax_base(wave_max(logit));
    w = used ? exp((double)logit - base) : 0;
    const double sum = p.normalize ? wave_sum(w) : total;
    w = nan ? __builtin_nan("") : sum == 0 ? 0 : w / sum;
  }
  if (used) {
    p.weights[t * p.k + lane] = (float)(w * p.scale);
    p.chosen[t * p.k + lane] = mine;
  }
}

template <class E, int PER>
__global__ void __launch_bounds__(256) route_kernel(RouteParams p) {
  __shared__ double s_score[4][PER * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t t = (int64_t)blockIdx.x * 4 + wave; t < p.tokens; t += (int64_t)gridDim.x * 4)
    route_token<E, PER>(p, t, lane, s_score[wave]);
}

// Gradient of the logits through the chosen scores.  One token a wave; a lane of the first k holds a chosen expert.
template <class E, int PER>
__device__ __forceinline__ void route_token_backward(const RouteParams& p, int64_t t, int lane, float* s_row) {
  const typename E::raw* x = static_cast<const typename E::raw*>(p.logits) + t * p.ldl;
  typename E::raw* dx = static_cast<typename E::raw*>(p.dlogits) + t * p.experts;
  const int e = lane < p.k ? p.chosen[t * p.k + lane] : -1;
  const bool used = e >= 0 && e < p.experts;
  const double dw = used ? (double)p.dweights[t * p.k + lane] * p.scale : 0;
  const float logit = used ? to_float<E>(x[e]) : -__builtin_inff();
  double s, mean = 0, base = 0, total = 1;
  const bool dense = !p.sigmoid && !p.normalize;
  if (p.sigmoid) {
    s = used ? sigmoid64(logit) : 0;
    const double slope = s * (1 - s);
    if (p.normalize) {
      total = wave_sum(s);
      mean = wave_sum(s * dw);
      s = total == 0 ? 0 : (dw - mean / total) / total * slope;
    } else {
      s = dw * slope;
    }
  } else {
    if (dense) {
      float top = -__builtin_inff();
      for (int i = lane; i < p.experts; i += 64) top = fmaxf(top, to_float<E>(x[i]));
      base = softmax_base(wave_max(top));
      total = 0;
      for (int i = lane; i < p.experts; i += 64) total += exp((double)to_float<E>(x[i]) - base);
      total = wave_sum(total);
    } else {
      base = softmax_base(wave_max(logit));
    }
    s = used ? exp((double)logit - base) : 0;
    if (!dense) total = wave_sum(s);
    s = total == 0 ? 0 : s / total;
    mean = wave_sum(s * dw);
    s *= dense ? dw : dw - mean;
  }
  for (int i = lane; i < p.experts; i += 64)
    s_row[i] = dense && total != 0 ? (float)(-mean * (exp((double)to_float<E>(x[i]) - base) / total)) : 0.0f;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if (used) s_row[e] += (float)s;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  for (int i = lane; i < p.experts; i += 64) dx[i] = from_float<E>(s_row[i]);
}

template <class E, int PER>
__global__ void __launch_bounds__(256) route_backward_kernel(RouteParams p) {
  __shared__ float s_row[4][PER * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t t = (int64_t)blockIdx.x * 4 + wave; t < p.tokens; t += (int64_t)gridDim.x * 4)
    route_token_backward<E, PER>(p, t, lane, s_row[wave]);
}

struct SortParams {
  const int32_t* experts;  // [n]
  int32_t* offs;           // [count]
  int32_t* slots;          // [n]
  int32_t* places;         // [n]
  int32_t* counts;         // workspace [blocks][count]
  int32_t n, first, count, chunk;  // chunk: entries of a workgroup, a multiple of 256
};

__device__ __forceinline__ int local_expert(const SortParams& p, int64_t i) {
  if (i >= p.n) return -1;
  const int64_t e = (int64_t)p.experts[i] - p.first;
  return e >= 0 && e < p.count ? (int)e : -1;
}

// How often each expert occurs in a workgroup's chunk.
__global__ void __launch_bounds__(256) sort_count_kernel(SortParams p) {
  __shared__ int32_t s_count[kSortExperts];
  for (int e = threadIdx.x; e < p.count; e += 256) s_count[e] = 0;
  __syncthreads();
  const int64_t begin = (int64_t)blockIdx.x * p.chunk;
  for (int i = threadIdx.x; i < p.chunk; i += 256) {
    const int e = local_expert(p, begin + i);
    if (e >= 0) atomicAdd(&s_count[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.count; e += 256) p.counts[(int64_t)blockIdx.x * p.count + e] = s_count[e];
}

// Places of a workgroup's chunk: behind the smaller experts, the earlier workgroups and waves, and the wave's own earlier
// entries, which it finds 64 at a time by matching the experts' bits across its lanes.  Counts are sums of integers and
// every order is that of the entries, so the result is the same at every call.
__global__ void __launch_bounds__(256) sort_place_kernel(SortParams p) {
  __shared__ int32_t s_next[4][kSortExperts];
  __shared__ int32_t s_part[256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t begin = (int64_t)blockIdx.x * p.chunk;
  const int span = p.chunk / 4;
  for (int e = threadIdx.x; e < 4 * kSortExperts; e += 256) (&s_next[0][0])[e] = 0;
  __syncthreads();
  for (int i = lane; i < span; i += 64) {
    const int e = local_expert(p, begin + wave * span + i);
    if (e >= 0) atomicAdd(&s_next[wave][e], 1);
  }
  // Four consecutive experts a thread: their counts in all workgroups and in the earlier ones.
  int total[4] = {}, before[4] = {}, sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = threadIdx.x * 4 + i;
    if (e < p.count)
      for (int b = 0; b < (int)gridDim.x; ++b) {
        const int n = p.counts[(int64_t)b * p.count + e];
        total[i] += n;
        before[i] += b < (int)blockIdx.x ? n : 0;
      }
    sum += total[i];
  }
  s_part[threadIdx.x] = sum;
  __syncthreads();
  for (int d = 1; d < 256; d <<= 1) {
    const int below = (int)threadIdx.x >= d ? s_part[threadIdx.x - d] : 0;
    __syncthreads();
    s_part[threadIdx.x] += below;
    __syncthreads();
  }
  int at = s_part[threadIdx.x] - sum;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = threadIdx.x * 4 + i;
    if (e >= p.count) break;
    int next = at + before[i];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int n = s_next[w][e];
      s_next[w][e] = next;
      next += n;
    }
    at += total[i];
    if (blockIdx.x == 0) p.offs[e] = at;
  }
  __syncthreads();
  const int used = s_part[255];
  const int bits = 32 - __builtin_clz((unsigned)p.count);
  for (int i = 0; i < span; i += 64) {
    const int64_t from = begin + wave * span + i + lane;
    const int e = local_expert(p, from);
    uint64_t same = __ballot(e >= 0);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? set : ~set;
    }
    int base = 0;
    const int leader = e >= 0 ? __builtin_ctzll(same) : lane;
    if (e >= 0 && lane == leader) base = atomicAdd(&s_next[wave][e], __builtin_popcountll(same));
    base = __shfl(base, leader);
    const int place = e >= 0 ? base + __builtin_popcountll(same & ((1ull << lane) - 1)) : -1;
    if (from < p.n) p.places[from] = place;
    if (place >= 0) p.slots[place] = (int32_t)from;
  }
  for (int i = threadIdx.x; i < p.chunk; i += 256)  // rows behind the last expert's
    if (begin + i >= used && begin + i < p.n) p.slots[begin + i] = -1;
}

struct RowsParams {
  const char* from;        // gather: tokens; combine and its gradient: sorted rows
  char* to;                // gather: sorted rows; combine: tokens; gradient: dy or null
  const int32_t* places;   // [tokens, k]
  const int32_t* end;      // the last offset
  const float* weights;    // [tokens, k] or null (1)
  const char* dout;        // gradient: [tokens, width]
  float* dweights;         // gradient: [tokens, k] or null
  int64_t ld_from, ld_to, ld_dout;  // bytes
  int64_t tokens;
  int32_t k, rows, width, spans;    // width in bytes; spans of a row
};

// Rows that no token went to are zeros.
template <class U>
__device__ __forceinline__ void clear_rows(const RowsParams& p, int block, int blocks) {
  const int used = min(max(*p.end, 0), p.rows);
  for (int64_t r = used + block; r < p.rows; r += blocks)
    for (int c = threadIdx.x * (int)sizeof(U); c < p.width; c += 256 * (int)sizeof(U))
      *reinterpret_cast<U*>(p.to + r * p.ld_to + c) = U{};
}

constexpr int kClearBlocks = 256;

// A wave copies up to SPAN x 64 units of one token to all its places: a token is read once.
template <class U>
__global__ void __launch_bounds__(256) gather_rows_kernel(RowsParams p) {
  constexpr int SPAN = 4;
  if (blockIdx.x < kClearBlocks) return clear_rows<U>(p, blockIdx.x, kClearBlocks);
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)(gridDim.x - kClearBlocks) * 4;
  for (int64_t item = ((int64_t)blockIdx.x - kClearBlocks) * 4 + (threadIdx.x >> 6); item < p.tokens * p.spans; item += waves) {
    const int64_t t = item / p.spans;
    const int64_t c0 = ((item - t * p.spans) * SPAN * 64 + lane) * (int64_t)sizeof(U);
    U v[SPAN];
#pragma unroll
    for (int u = 0; u < SPAN; ++u) {
      const int64_t c = c0 + u * 64 * sizeof(U);
      if (c < p.width) v[u] = *reinterpret_cast<const U*>(p.from + t * p.ld_from + c);
    }
    for (int j = 0; j < p.k; ++j) {
      const int place = p.places[t * p.k + j];
      if (place < 0 || place >= p.rows) continue;
#pragma unroll
      for (int u = 0; u < SPAN; ++u) {
        const int64_t c = c0 + u * 64 * sizeof(U);
        if (c < p.width) *reinterpret_cast<U*>(p.to + (int64_t)place * p.ld_to + c) = v[u];
      }
    }
  }
}

// N elements of a unit as fp32 and back.
template <class E, class U>
struct Unit {
  static constexpr int N = sizeof(U) / sizeof(typename E::raw);
  static __device__ __forceinline__ void widen(const U& u, float (&v)[N]) {
    typename E::raw r[N];
    __builtin_memcpy(r, &u, sizeof(U));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_float<E>(r[i]);
  }
  static __device__ __forceinline__ U narrow(const float (&v)[N]) {
    typename E::raw r[N];
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = from_float<E>(v[i]);
    U u;
    __builtin_memcpy(&u, r, sizeof(U));
    return u;
  }
};

// A wave sums one span of a token's rows in the order of its slots, in fp32, and rounds once.
template <class E, class U>
__global__ void __launch_bounds__(256) combine_rows_kernel(RowsParams p) {
  using Q = Unit<E, U>;
  constexpr int SPAN = 2;
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * 4;
  for (int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); item < p.tokens * p.spans; item += waves) {
    const int64_t t = item / p.spans;
    const int64_t c0 = ((item - t * p.spans) * SPAN * 64 + lane) * (int64_t)sizeof(U);
    float sum[SPAN][Q::N] = {};
    for (int j = 0; j < p.k; ++j) {
      const int place = p.places[t * p.k + j];
      if (place < 0 || place >= p.rows) continue;
      const float w = p.weights ? p.weights[t * p.k + j] : 1.0f;
#pragma unroll
      for (int u = 0; u < SPAN; ++u) {
        const int64_t c = c0 + u * 64 * sizeof(U);
        if (c >= p.width) continue;
        float v[Q::N];
        Q::widen(*reinterpret_cast<const U*>(p.from + (int64_t)place * p.ld_from + c), v);
#pragma unroll
        for (int i = 0; i < Q::N; ++i) sum[u][i] += w * v[i];
      }
    }
#pragma unroll
    for (int u = 0; u < SPAN; ++u) {
      const int64_t c = c0 + u * 64 * sizeof(U);
      if (c < p.width) *reinterpret_cast<U*>(p.to + t * p.ld_to + c) = Q::narrow(sum[u]);
    }
  }
}

// One routed row a wave: dy = w dout and dw = <dout, y>, the product's sum over its lanes in one fixed order.
template <class E, class U>
__global__ void __launch_bounds__(256) combine_rows_backward_kernel(RowsParams p) {
  using Q = Unit<E, U>;
  if (blockIdx.x < kClearBlocks) {
    if (p.to) clear_rows<U>(p, blockIdx.x, kClearBlocks);
    return;
  }
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)(gridDim.x - kClearBlocks) * 4;
  for (int64_t slot = ((int64_t)blockIdx.x - kClearBlocks) * 4 + (threadIdx.x >> 6); slot < p.tokens * p.k; slot += waves) {
    const int place = p.places[slot];
    const bool here = place >= 0 && place < p.rows;
    float dot = 0;
    if (here) {
      const char* dout = p.dout + slot / p.k * p.ld_dout;
      const float w = p.weights ? p.weights[slot] : 1.0f;
      for (int64_t c = lane * (int)sizeof(U); c < p.width; c += 64 * sizeof(U)) {
        float d[Q::N], y[Q::N];
        Q::widen(*reinterpret_cast<const U*>(dout + c), d);
        if (p.dweights) {
          Q::widen(*reinterpret_cast<const U*>(p.from + (int64_t)place * p.ld_from + c), y);
#pragma unroll
          for (int i = 0; i < Q::N; ++i) dot += d[i] * y[i];
        }
        if (p.to) {
#pragma unroll
          for (int i = 0; i < Q::N; ++i) d[i] *= w;
          *reinterpret_cast<U*>(p.to + (int64_t)place * p.ld_to + c) = Q::narrow(d);
        }
      }
    }
    if (p.dweights) {
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) dot += __shfl_xor(dot, d);
      if (lane == 0) p.dweights[slot] = dot;
    }
  }
}

}  // namespace moegemm
