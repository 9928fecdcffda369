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

// One token a wave, on 64-bit scores, so that which of two close ones is larger never hangs on a rounding of exp.  The keys
// lie in LDS (two arrays of the experts' number): the loops are short and hold few registers.
template <class E>
__device__ void route_token(const RouteParams& p, int64_t t, int lane, uint64_t* key, uint64_t* group) {
  const typename E::raw* x = static_cast<const typename E::raw*>(p.logits) + t * p.ldl;
  float top = -__builtin_inff();
  bool nan = false;
  for (int e = lane; e < p.experts; e += 64) {
    const float v = to_float<E>(x[e]);
    nan |= v != v;
    top = fmaxf(top, v);
  }
  nan = __ballot(nan) != 0;
  // Without a bias, and unless scores are added up, they rank as the logits do.
  const bool by_logit = !p.bias && p.group_best == 1;
  float base = 0;
  double total = 1;
  if (!p.sigmoid) {
    base = softmax_base(wave_max(top));
    total = 0;
    for (int e = lane; e < p.experts; e += 64) total += exp((double)to_float<E>(x[e]) - base);
    total = wave_sum(total);
  }
  for (int e = lane; e < p.experts; e += 64) {
    const double v = to_float<E>(x[e]);
    double c = v;
    if (!by_logit) c = p.sigmoid ? sigmoid64(v) : total == 0 ? 0 : exp(v - base) / total;
    key[e] = order_of(p.bias ? c + p.bias[e] : c);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  auto take = [&](uint64_t* keys, int count) {  // the best of them, struck out
    Best b{0, 0};
    for (int i = lane; i < count; i += 64) better(b, keys[i], i);
    b = wave_best(b);
    if (lane == 0) keys[b.index] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return b.index;
  };
  if (p.groups > 1) {
    const int size = p.experts / p.groups;
    auto score_of = [](uint64_t k) {
      return k == 1 ? __builtin_nan("") : __builtin_bit_cast(double, k >> 63 ? k ^ (1ull << 63) : ~k);
    };
    for (int g = lane; g < p.groups; g += 64) {
      uint64_t first = 0, second = 0;
      for (int e = 0; e < size; ++e) {
        const uint64_t c = key[g * size + e];
        if (c > first) {
          second = first;
          first = c;
        } else if (c > second) {
          second = c;
        }
      }
      group[g] = order_of(p.group_best == 2 && size > 1 ? score_of(first) + score_of(second) : score_of(first));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int n = 0; n < p.top_groups; ++n) take(group, p.groups);  // kept groups are 0 now
    for (int e = lane; e < p.experts; e += 64)
      if (group[e / size] != 0) key[e] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  int mine = 0;
  for (int j = 0; j < p.k; ++j) {
    const int e = take(key, p.experts);
    if (lane == j) mine = e;
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

// Lanes of a token: rows of 16 lanes exchange values at full rate (DPP), the wave's four rows in two more steps.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140, kRor = 0x120;  // quad_perm, row_*

// f over the LPT lanes of a token, f commutative and associative.
template <int LPT, class F>
__device__ __forceinline__ uint32_t token_reduce(uint32_t x, F&& f) {
  x = f(x, dpp<kXor1>(x));
  x = f(x, dpp<kXor2>(x));
  x = f(x, dpp<kHalfMirror>(x));
  x = f(x, dpp<kMirror>(x));
  if constexpr (LPT == 64) {
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = f(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = f(b[0], b[1]);
  }
  return x;
}
template <int LPT>
__device__ __forceinline__ uint32_t token_max(uint32_t x) {
  return token_reduce<LPT>(x, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int LPT>
__device__ __forceinline__ float token_max(float x) {
  return __builtin_bit_cast(float, token_reduce<LPT>(__builtin_bit_cast(uint32_t, x), [](uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
  }));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint64_t lo = dpp<CTRL>((uint32_t)u), hi = dpp<CTRL>((uint32_t)(u >> 32));
  return __builtin_bit_cast(double, hi << 32 | lo);
}
template <int LPT>
__device__ __forceinline__ double token_sum(double x) {
  x += dpp<kXor1>(x);
  x += dpp<kXor2>(x);
  x += dpp<kHalfMirror>(x);
  x += dpp<kMirror>(x);
  if constexpr (LPT == 64) {
    x += __shfl_xor(x, 16);
    x += __shfl_xor(x, 32);
  }
  return x;
}

__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float score_of(uint32_t key) {
  return __builtin_bit_cast(float, key >> 31 ? key ^ 0x80000000u : ~key);
}
// Whether fp32 scores a >= b, each within 2^-20 (1 + its size) of the exact one, cut below by up to 16 units, may stand in
// the wrong order (or one of them is no number).  An exp of |x| 2^-24 relative error costs sigmoid and softmax at most 2^-22, a
// sum of up to 1024 exps by 16 + 6 additions 2^-19 of a softmax.
__device__ __forceinline__ bool too_close(float a, float b, float margin) {
  return !(a - b > margin * fmaxf(1.0f, fmaxf(fabsf(a), fabsf(b))));
}
constexpr float kRouteMargin = 0x1p-17f;

// 64 / LPT tokens a wave, expert lane * per + i.  Scores are taken in fp32 and compared as integers whose lowest bits tell a
// lane's experts apart; tokens with two scores too close for that to be sure of go to route_token, one after the
// other.  Normal scores send one token in some hundred there.  16-bit logits that rank by themselves leave 13 bits free, which
// hold the whole index: their order is exact, and equal ones are no reason.
//
// Bound by the vector instructions: the k rounds of a maximum over PER registers and LPT lanes.
template <class E, int LPT, int PER>
__global__ void __launch_bounds__(256) route_kernel(RouteParams p) {
  constexpr int TOKENS = 64 / LPT;
  constexpr uint32_t MASK = PER - 1, WHOLE = 0x1fff;
  extern __shared__ uint64_t s_key[];  // route_token's arrays, for each wave
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int li = lane & (LPT - 1), sub = lane / LPT;
  const int per = (p.experts + LPT - 1) / LPT, e0 = li * per;
  uint64_t* keys = s_key + wave * (p.experts + p.groups);
  const bool by_logit = !p.bias && p.group_best == 1;
  const bool whole = by_logit && !E::is_f32;
  const bool needs_total = !p.sigmoid && !p.normalize;
  const bool vec = per == PER && PER * sizeof(typename E::raw) % 16 == 0 && p.experts == LPT * PER &&
                   (reinterpret_cast<uintptr_t>(p.logits) & 15) == 0 && p.ldl * sizeof(typename E::raw) % 16 == 0;
  const int group_lanes = LPT / p.groups;  // the caller's promise where groups > 1: see fast_route
  float bias[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) bias[i] = p.bias && i < per && e0 + i < p.experts ? p.bias[e0 + i] : 0.0f;

  const int64_t step = (int64_t)gridDim.x * 4 * TOKENS;
  for (int64_t t0 = ((int64_t)blockIdx.x * 4 + wave) * TOKENS; t0 < p.tokens; t0 += step) {
    const int64_t t = min(t0 + sub, (int64_t)p.tokens - 1);  // a wave's missing tokens repeat the last one
    const typename E::raw* x = static_cast<const typename E::raw*>(p.logits) + t * p.ldl;
    float v[PER];
    if (vec) {
      typename E::raw raw[PER];
      constexpr int N = PER * sizeof(typename E::raw) / 16;
      u32x4_t c[N > 0 ? N : 1];
#pragma unroll
      for (int i = 0; i < N; ++i) c[i] = reinterpret_cast<const u32x4_t*>(x + e0)[i];
      __builtin_memcpy(raw, c, N > 0 ? sizeof(raw) : 0);
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] = to_float<E>(raw[i]);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] = i < per && e0 + i < p.experts ? to_float<E>(x[e0 + i]) : -__builtin_inff();
    }
    bool doubt = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) doubt |= v[i] != v[i];
    float c[PER];
    double total = 1;
    float base = 0;
    if (needs_total || (!p.sigmoid && !by_logit)) {
      float top = v[0];
#pragma unroll
      for (int i = 1; i < PER; ++i) top = fmaxf(top, v[i]);
      base = softmax_base(token_max<LPT>(top));
    }
    if (needs_total) {
      total = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (i < per) total += exp((double)v[i] - base);
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // four at a time: sixteen side by side take all registers
      }
      total = token_sum<LPT>(total);
    }
    if (by_logit) {
#pragma unroll
      for (int i = 0; i < PER; ++i) c[i] = v[i];
    } else if (p.sigmoid) {
#pragma unroll
      for (int i = 0; i < PER; ++i) c[i] = __builtin_amdgcn_rcpf(1.0f + __expf(-v[i])) + bias[i];
    } else {
      double sum = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        c[i] = __expf(v[i] - base);
        sum += c[i];
      }
      const float inverse = (float)(1.0 / token_sum<LPT>(sum));
#pragma unroll
      for (int i = 0; i < PER; ++i) c[i] = c[i] * inverse + bias[i];
    }
    bool mine_in = true;  // a lane's experts are of one group
    if (p.groups > 1) {
      float first = -__builtin_inff(), second = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i < per) {
          second = fmaxf(second, fminf(first, c[i]));
          first = fmaxf(first, c[i]);
        }
      auto merge = [&](float f, float s) {
        second = fmaxf(fminf(first, f), fmaxf(second, s));
        first = fmaxf(first, f);
      };
      // Row by row: groups of 2, 4, 8 or 16 lanes; 64 lanes have groups of 4 or more.
      auto bits = [](float f) { return __builtin_bit_cast(uint32_t, f); };
      auto real = [](uint32_t u) { return __builtin_bit_cast(float, u); };
      if (group_lanes >= 2) merge(real(dpp<kXor1>(bits(first))), real(dpp<kXor1>(bits(second))));
      if (group_lanes >= 4) merge(real(dpp<kXor2>(bits(first))), real(dpp<kXor2>(bits(second))));
      if (group_lanes >= 8) merge(real(dpp<kHalfMirror>(bits(first))), real(dpp<kHalfMirror>(bits(second))));
      if (group_lanes >= 16) merge(real(dpp<kMirror>(bits(first))), real(dpp<kMirror>(bits(second))));
      if (LPT == 64 && group_lanes >= 32) merge(__shfl_xor(first, 16), __shfl_xor(second, 16));
      const float score = p.group_best == 2 && p.experts > p.groups ? first + second : first;
      int rank = 0;
      for (int g = 1; g < p.groups; ++g) {
        const int from = (lane & ~(LPT - 1)) | ((li + g * group_lanes) & (LPT - 1));
        const float other = __shfl(score, from);
        rank += other > score || (other == score && (from & (LPT - 1)) < li) ? 1 : 0;
      }
      mine_in = rank < p.top_groups;
      if (p.top_groups < p.groups) {
        const float least = -token_max<LPT>(mine_in ? -score : -__builtin_inff());
        const float most = token_max<LPT>(mine_in ? -__builtin_inff() : score);
        doubt |= too_close(least, most, 2 * kRouteMargin);
      }
    }
    uint32_t key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t low = whole ? WHOLE - (uint32_t)(e0 + i) : MASK - (uint32_t)i;
      const uint32_t o = (order_of(c[i]) & ~(whole ? WHOLE : MASK)) | low;
      key[i] = i < per && e0 + i < p.experts && mine_in ? o : 0;
    }
    int mine = 0;
    float last = 0;
    for (int j = 0; j <= p.k; ++j) {
      uint32_t top = key[0];
#pragma unroll
      for (int i = 1; i < PER; ++i) top = max(top, key[i]);
      const uint32_t best = token_max<LPT>(top);
      const float score = score_of(best & ~MASK);
      if (!whole && j > 0 && best) doubt |= too_close(last, score, kRouteMargin);
      last = score;
      if (j == p.k) break;
      uint64_t hits = __ballot(top == best);
      if constexpr (LPT == 16) hits = hits >> (lane & 48) & 0xffff;
      doubt |= !whole && (hits & (hits - 1)) != 0;
      const int e = whole ? (int)(WHOLE - (best & WHOLE)) : (int)__builtin_ctzll(hits) * per + (int)(MASK - (best & MASK));
      if (li == j) mine = min(e, p.experts - 1);
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = key[i] == best ? 0 : key[i];
    }
    const uint64_t doubts = __ballot(doubt);
    const bool used = li < p.k;
    const float logit = used ? to_float<E>(x[mine]) : -__builtin_inff();
    double w;
    if (p.sigmoid) {
      w = used ? sigmoid64(logit) : 0;
      if (p.normalize) {
        const double sum = token_sum<LPT>(w);
        w = sum == 0 ? 0 : w / sum;
      }
    } else {
      if (p.normalize) base = softmax_base(token_max<LPT>(logit));
      w = used ? exp((double)logit - base) : 0;
      if (p.normalize) total = token_sum<LPT>(w);
      w = total == 0 ? 0 : w / total;
    }
    constexpr uint64_t LANES = LPT == 64 ? ~0ull : (1ull << (LPT & 63)) - 1;
    if (used && t0 + sub < p.tokens && (doubts >> (sub * LPT) & LANES) == 0) {
      p.weights[t * p.k + li] = (float)(w * p.scale);
      p.chosen[t * p.k + li] = mine;
    }
    if (doubts == 0) continue;
    for (int n = 0; n < TOKENS; ++n)
      if (t0 + n < p.tokens && (doubts >> (n * LPT) & LANES) != 0) route_token<E>(p, t0 + n, lane, keys, keys + p.experts);
  }
}

// Every token on 64-bit scores, one a wave: more than 64 experts to choose in rows of 16 lanes, or groups that lanes cannot hold.
template <class E>
__global__ void __launch_bounds__(256) route_exact_kernel(RouteParams p) {
  extern __shared__ uint64_t s_key[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t* keys = s_key + wave * (p.experts + p.groups);
  for (int64_t t = (int64_t)blockIdx.x * 4 + wave; t < p.tokens; t += (int64_t)gridDim.x * 4)
    route_token<E>(p, t, lane, keys, keys + p.experts);
}

// Gradient of the logits through the chosen scores.  64 / LPT tokens a wave; a lane of a token's first k holds a chosen expert.
// Where the gradient is not dense it is k numbers among zeros, put together in LDS and stored in whole lines.
template <class E, int LPT, int PER>
__global__ void __launch_bounds__(256) route_backward_kernel(RouteParams p) {
  constexpr int TOKENS = 64 / LPT;
  __shared__ __attribute__((aligned(16))) float s_row[4][TOKENS][LPT * PER];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int li = lane & (LPT - 1), sub = lane / LPT;
  const bool dense = !p.sigmoid && !p.normalize;
  float* row = s_row[wave][sub];
  const int64_t step = (int64_t)gridDim.x * 4 * TOKENS;
  for (int64_t t0 = ((int64_t)blockIdx.x * 4 + wave) * TOKENS; t0 < p.tokens; t0 += step) {
    const int64_t t = min(t0 + sub, (int64_t)p.tokens - 1);
    const typename E::raw* x = static_cast<const typename E::raw*>(p.logits) + t * p.ldl;
    const int e = li < p.k ? p.chosen[t * p.k + li] : -1;
    const bool used = e >= 0 && e < p.experts;
    const double dw = used ? (double)p.dweights[t * p.k + li] * p.scale : 0;
    const float logit = used ? to_float<E>(x[e]) : -__builtin_inff();
    double s;
    if (p.sigmoid) {
      s = used ? sigmoid64(logit) : 0;
      const double slope = s * (1 - s);
      if (p.normalize) {
        const double total = token_sum<LPT>(s), mean = token_sum<LPT>(s * dw);
        s = total == 0 ? 0 : (dw - mean / total) / total * slope;
      } else {
        s = dw * slope;
      }
    } else if (dense) {
      double all[PER], total = 0;
      float v[PER], top = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        v[i] = li + i * LPT < p.experts ? to_float<E>(x[li + i * LPT]) : -__builtin_inff();
        top = fmaxf(top, v[i]);
      }
      const float base = softmax_base(token_max<LPT>(top));
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        all[i] = li + i * LPT < p.experts ? exp((double)v[i] - base) : 0;
        total += all[i];
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
      total = token_sum<LPT>(total);
      const double inverse = total == 0 ? 0 : 1 / total;
      s = used ? exp((double)logit - base) * inverse * dw : 0;
      const double mean = token_sum<LPT>(s);
#pragma unroll
      for (int i = 0; i < PER; ++i) row[li + i * LPT] = (float)(-mean * (all[i] * inverse));
    } else {
      const float base = softmax_base(token_max<LPT>(logit));
      s = used ? exp((double)logit - base) : 0;
      const double total = token_sum<LPT>(s);
      s = total == 0 ? 0 : s / total;
      s *= dw - token_sum<LPT>(s * dw);
    }
    if (!dense) {
#pragma unroll
      for (int i = 0; i < PER; ++i) row[li + i * LPT] = 0;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (used) row[e] += (float)s;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    // The rows of the wave's tokens one after the other, 16 bytes a lane where they allow it.
    constexpr int N = 16 / sizeof(typename E::raw);
    const bool vec = p.experts % N == 0 && (reinterpret_cast<uintptr_t>(p.dlogits) & 15) == 0;
    for (int n = 0; n < TOKENS; ++n) {
      if (t0 + n >= p.tokens) break;
      typename E::raw* dx = static_cast<typename E::raw*>(p.dlogits) + (t0 + n) * p.experts;
      const float* from = s_row[wave][n];
      if (vec) {
        for (int i = lane * N; i < p.experts; i += 64 * N) {
          typename E::raw out[N];
#pragma unroll
          for (int j = 0; j < N; ++j) out[j] = from_float<E>(from[i + j]);
          u32x4_t packed;
          __builtin_memcpy(&packed, out, 16);
          *MOEGEMM_GLOBAL(u32x4_t, dx + i) = packed;
        }
      } else {
        for (int i = lane; i < p.experts; i += 64) dx[i] = from_float<E>(from[i]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // read before the next tokens' rows are written
  }
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
