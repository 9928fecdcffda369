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

#include <type_traits>

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

typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

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

// Scores as integers of the same order; a NaN lies below -inf, and 0 below everything is "not to be had".  -0 + 0 is 0:
// zeros of both signs are one score.
__device__ __forceinline__ uint64_t order_of(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);
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

// One token a wave, on 64-bit scores, so that which of two close ones is larger never hangs on a rounding of exp.  The
// keys lie in LDS (two arrays of the experts' number): the loops are short and hold few registers.
template <class E>
__device__ __forceinline__ void route_token(const RouteParams& p, int64_t t, int lane, uint64_t* key, uint64_t* group) {
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
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float score_of(uint32_t key) {
  return __builtin_bit_cast(float, key >> 31 ? key ^ 0x80000000u : ~key);
}
// fp32 scores are within 2^-22 of sigmoid (exp of x is off by (|x| + 2) 2^-24 of itself, the sum and the reciprocal by
// 2^-24 and 2^-23, and s (1 - s) |x| < 1/4) and of softmax (whose sum is a 64-bit one, and |x| e^-|x| < 0.4); a bias
// adds 2^-24 of the sum. Keys drop up to `mask` units of 2^-23 of their size.  Scores further apart than this, times
// their size or 1, are in order; sums of two than twice this, times the size of the largest term or 1 (the terms' errors,
// 2^-21 and 2^-22 of their size with the sum's rounding, of either sum).
__host__ __device__ constexpr float route_margin(uint32_t mask) { return (float)(mask + 1) * 0x1p-23f + 0x1p-20f; }

// Whether a, the larger in fp32, may not be the larger one (or is no number).
__device__ __forceinline__ bool too_close(double a, double b, double margin) {
  return !(a - b > margin * fmax(1.0, fmax(fabs(a), fabs(b))));
}

// The two largest of a token's group, GROUP lanes with their own two largest.
template <class F, class M>
__device__ __forceinline__ void group_two(F& first, F& second, int group_lanes, bool wide, M&& row) {
  auto merge = [&](F f, F s) {
    second = fmax(fmin(first, f), fmax(second, s));
    first = fmax(first, f);
  };
  if (group_lanes >= 2) merge(row(first, std::integral_constant<int, kXor1>{}), row(second, std::integral_constant<int, kXor1>{}));
  if (group_lanes >= 4) merge(row(first, std::integral_constant<int, kXor2>{}), row(second, std::integral_constant<int, kXor2>{}));
  if (group_lanes >= 8)
    merge(row(first, std::integral_constant<int, kHalfMirror>{}), row(second, std::integral_constant<int, kHalfMirror>{}));
  if (group_lanes >= 16)
    merge(row(first, std::integral_constant<int, kMirror>{}), row(second, std::integral_constant<int, kMirror>{}));
  if (wide && group_lanes >= 32) merge(__shfl_xor(first, 16), __shfl_xor(second, 16));
}

// Descending order of N registers by compare and exchange: runs that fall and rise in turn, merged to twice their
// length.
template <int N>
__device__ __forceinline__ void sort_descending(uint32_t (&a)[N]) {
#pragma unroll
  for (int k = 2; k <= N; k *= 2)
#pragma unroll
    for (int j = k / 2; j > 0; j /= 2)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (!(i & j)) {
          const uint32_t x = a[i], y = a[i + j];
          const bool falls = (i & k) == 0 || k == N;
          a[i] = falls ? max(x, y) : min(x, y);
          a[i + j] = falls ? min(x, y) : max(x, y);
        }
}
// The same where a rises and then falls, or falls and then rises.
template <int N>
__device__ __forceinline__ void merge_descending(uint32_t (&a)[N]) {
#pragma unroll
  for (int j = N / 2; j > 0; j /= 2)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (!(i & j)) {
        const uint32_t x = a[i], y = a[i + j];
        a[i] = max(x, y);
        a[i + j] = min(x, y);
      }
}
// Each lane's list becomes the largest N of its own and its partner's: both fall, so the larger of one from the front
// and one from the back are those.
template <int CTRL, int N>
__device__ __forceinline__ void join_lists(uint32_t (&a)[N]) {
  uint32_t b[N];
#pragma unroll
  for (int i = 0; i < N; ++i) b[i] = max(a[i], (uint32_t)__builtin_amdgcn_mov_dpp((int)a[N - 1 - i], CTRL, 0xf, 0xf, true));
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = b[i];
  merge_descending(a);
}
template <bool HALVES, int N>
__device__ __forceinline__ void join_lists_across(uint32_t (&a)[N]) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    // swap(x, y) leaves (x0, y0) and (x1, y1) of the two rows (halves).
    const uint32_t x = a[i], y = a[N - 1 - i];
    const auto f = HALVES ? __builtin_amdgcn_permlane32_swap(x, y, false, false) : __builtin_amdgcn_permlane16_swap(x, y, false, false);
    const auto g = HALVES ? __builtin_amdgcn_permlane32_swap(y, x, false, false) : __builtin_amdgcn_permlane16_swap(y, x, false, false);
    a[i] = max(f[0], g[1]);
    a[N - 1 - i] = max(g[0], f[1]);
  }
  merge_descending(a);
}

// 64 / LPT tokens a wave, expert lane * per + i.  Scores are taken in fp32 as integers whose lowest bits name the
// expert; each lane sorts its own, and the lanes' lists are joined to the token's TOP best, which every lane then
// holds: compares and exchanges between registers, with no round of a maximum for each of the k.  Where two scores are
// too close for their order to be sure of, those in question are taken again in 64 bits: the groups', and of the TOP
// best the order.  What even that leaves open (a NaN, or the k-th too close to what is not on the list) goes to
// route_token, one token after the other.  16-bit logits that rank by themselves leave 13 bits free: their order is
// exact, and equal ones are in order.
//
// Bound by the vector instructions: 320 a token of 256 experts with groups, 7 tenths of the busy cycles, and 9 tenths of 896
// experts.  16384 tokens, 8 of 256 experts, fp32: by their logits 9.5 us, by sigmoid with a bias 11.1, 4 of 8 groups too
// 13.3 to 15.4, by how many are close (1.1 TB/s of logits); 4097 tokens, 16 of 896 bf16 by softmax unnormalised 17.3; one
// token 4.7, a launch and the chain of its steps.  Softmax scores with a bias pay for closeness most, since the margin is
// that of scores up to 1: 16384 x 256 of logits N(0, 1.5) 16.8, of N(0, 0.02), a router that has not learnt yet, 77 (one
// token after the other; by route_exact_kernel 47).
enum RouteRank {
  RANK_LOGITS,      // scores rank as the logits do
  RANK_LOGITS_SUM,  // and a softmax's sum over all experts is needed for the weights
  RANK_SIGMOID,
  RANK_SOFTMAX,
};
template <class E, int LPT, int PER, int TOP, RouteRank RANK>
__global__ void __launch_bounds__(256) route_kernel(RouteParams p) {
  using raw_t = typename E::raw;
  constexpr bool SCORES = RANK >= RANK_SIGMOID;
  constexpr int TOKENS = 64 / LPT;
  constexpr bool WHOLE = !SCORES && !E::is_f32;
  constexpr uint32_t MASK = WHOLE ? 0x1fff : LPT * PER - 1;
  constexpr uint64_t LANES = LPT == 64 ? ~0ull : (1ull << (LPT & 63)) - 1;
  extern __shared__ uint64_t s_key[];  // route_token's arrays, for each wave
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int li = lane & (LPT - 1), sub = lane / LPT, lane0 = lane & ~(LPT - 1);
  const int per = (p.experts + LPT - 1) / LPT, e0 = li * per;
  const int count = max(min(per, p.experts - e0), 0);  // the lane's experts
  const int group_lanes = LPT / p.groups;              // divides where groups > 1 (see fast_route)
  const bool vec = p.experts == LPT * PER && PER * sizeof(raw_t) % 16 == 0 &&
                   (reinterpret_cast<uintptr_t>(p.logits) & 15) == 0 && p.ldl * sizeof(raw_t) % 16 == 0;

  // No loop over tokens: it would hold the constants of exp in registers throughout.
  const int t0 = ((int)blockIdx.x * 4 + wave) * TOKENS;
  if (t0 < p.tokens) {
    const int64_t t = min(t0 + sub, p.tokens - 1);  // a wave's missing tokens repeat the last one
    const raw_t* x = static_cast<const raw_t*>(p.logits) + t * p.ldl;
    float c[PER];
    if (vec) {
      constexpr int N = PER * sizeof(raw_t) / 16;
      if constexpr (N > 0) {
        raw_t raw[PER];
        u32x4_t chunk[N];
#pragma unroll
        for (int i = 0; i < N; ++i) chunk[i] = reinterpret_cast<const u32x4_t*>(x + e0)[i];
        __builtin_memcpy(raw, chunk, sizeof(raw));
#pragma unroll
        for (int i = 0; i < PER; ++i) c[i] = to_float<E>(raw[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) c[i] = to_float<E>(x[min(e0 + i, p.experts - 1)]);  // no branch around a load
#pragma unroll
      for (int i = 0; i < PER; ++i) c[i] = i < count ? c[i] : -__builtin_inff();
    }
    bool lost = false;  // for route_token to settle
#pragma unroll
    for (int i = 0; i < PER; ++i) lost |= c[i] != c[i];
    double total = 1;
    float base = 0;
    if constexpr (RANK == RANK_LOGITS_SUM || RANK == RANK_SOFTMAX) {
      float top = c[0];
#pragma unroll
      for (int i = 1; i < PER; ++i) top = fmaxf(top, c[i]);
      base = softmax_base(token_max<LPT>(top));
      total = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (i < per) total += exp((double)c[i] - base);
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // four at a time: sixteen side by side take all registers
      }
      total = token_sum<LPT>(total);
    }
    // The score of an expert in 64 bits.
    auto score64 = [&](float logit, int e) {
      double s = logit;
      if constexpr (SCORES) s = RANK == RANK_SIGMOID ? sigmoid64(s) : total == 0 ? 0 : exp(s - base) / total;
      return SCORES && p.bias ? s + p.bias[e] : s;
    };
    if constexpr (SCORES) {
      if constexpr (RANK == RANK_SIGMOID) {
#pragma unroll
        for (int i = 0; i < PER; ++i) c[i] = __builtin_amdgcn_rcpf(1.0f + __expf(-c[i]));
      } else {
        const float inverse = total != 0 ? (float)(1 / total) : 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) c[i] = __expf(c[i] - base) * inverse;
      }
      if (p.bias) {
        if (vec) {
#pragma unroll
          for (int i = 0; i < PER; i += 4) {
            const f32x4_t b = *reinterpret_cast<const f32x4_a4*>(p.bias + e0 + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) c[i + j] += b[j];
          }
        } else {
#pragma unroll
          for (int i = 0; i < PER; ++i) c[i] += p.bias[min(e0 + i, p.experts - 1)];
        }
      }
    }
    if constexpr (SCORES) {
#pragma unroll
      for (int i = 0; i < PER; ++i) lost |= (int)(i < count) & (int)(c[i] != c[i]);
    }
    bool mine_in = true;  // a lane's experts are of one group
    if (p.groups > 1) {
      // A group's place among the groups: how many are before it.
      auto place = [&](auto score) {
        int rank = 0;
#pragma unroll
        for (int g = 1; g < 16; ++g) {
          const int from = lane0 | ((li + g * group_lanes) & (LPT - 1));
          const auto other = __shfl(score, from);
          rank += (int)(g < p.groups) & ((int)(other > score) | ((int)(other == score) & (int)(from < lane)));
        }
        return rank;
      };
      const bool two = p.group_best == 2 && p.experts > p.groups;
      float first = -__builtin_inff(), second = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const float each = i < per ? c[i] : -__builtin_inff();
        second = fmaxf(second, fminf(first, each));
        first = fmaxf(first, each);
      }
      group_two(first, second, group_lanes, LPT == 64, [](float f, auto ctrl) {
        return __builtin_bit_cast(float, dpp<decltype(ctrl)::value>(__builtin_bit_cast(uint32_t, f)));
      });
      const float score = two ? first + second : first;
      lost |= score != score;  // inf - inf
      mine_in = place(score) < p.top_groups;
      const float least = -token_max<LPT>(mine_in ? -score : -__builtin_inff());
      const float most = token_max<LPT>(mine_in ? -__builtin_inff() : score);
      // Terms that a bias made large and that cancel leave a sum as wrong as they are; an infinite one is exact.
      auto finite_size = [](float f) { return fabsf(f) < __builtin_inff() ? fabsf(f) : 0.0f; };
      const double size = token_max<LPT>(fmaxf(finite_size(first), two ? finite_size(second) : 0.0f));
      if (__ballot(p.top_groups < p.groups && !((double)least - most > 2 * route_margin(0) * fmax(1.0, size)))) {
        double first = -__builtin_inf(), second = -__builtin_inf();
#pragma unroll 1
        for (int i = 0; i < per; ++i) {
          const double each = score64(to_float<E>(x[e0 + i]), e0 + i);
          second = fmax(second, fmin(first, each));
          first = fmax(first, each);
        }
        group_two(first, second, group_lanes, LPT == 64, [](double f, auto ctrl) { return dpp<decltype(ctrl)::value>(f); });
        mine_in = place(two ? first + second : first) < p.top_groups;
      }
    }
    uint32_t key[PER], list[TOP] = {};
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t o = (order_of(c[i]) & ~MASK) | (MASK - (uint32_t)(e0 + i));
      key[i] = (int)(i < count) & (int)mine_in ? o : 0;
    }
    sort_descending(key);
#pragma unroll
    for (int i = 0; i < min(PER, TOP); ++i) list[i] = key[i];
    join_lists<kXor1>(list);
    join_lists<kXor2>(list);
    join_lists<kHalfMirror>(list);
    join_lists<kMirror>(list);
    if constexpr (LPT == 64) {
      join_lists_across<false>(list);
      join_lists_across<true>(list);
    }
    uint32_t own = 0, next = 0;  // the li-th best and the one behind it
#pragma unroll
    for (int i = 0; i < TOP; ++i) {
      own = li == i ? list[i] : own;
      next = li == i - 1 ? list[i] : next;
    }
    int mine = own ? (int)(MASK - (own & MASK)) : 0;
    float logit = own ? to_float<E>(x[mine]) : -__builtin_inff();
    if constexpr (!WHOLE) {
      const bool close = own != 0 && next != 0 && too_close(score_of(own & ~MASK), score_of(next & ~MASK), route_margin(MASK));
      if (__ballot(close && li < p.k)) {
        // The list's order by 64-bit scores; what is not on it has to be smaller than the k-th by more than its error.
        const double score = own ? score64(logit, mine) : -__builtin_inf();
        int rank = 0;
#pragma unroll 1
        for (int j = 0; j < TOP; ++j) {
          const double other = __shfl(score, lane0 + j);
          const int index = __shfl(own ? mine : 0x7fffffff, lane0 + j);
          rank += (int)(other > score) | ((int)(other == score) & (int)(index < mine));
        }
        const int to = (lane0 + (own ? rank : li)) * 4;
        mine = __builtin_amdgcn_ds_permute(to, mine);
        logit = __builtin_bit_cast(float, __builtin_amdgcn_ds_permute(to, __builtin_bit_cast(int, logit)));
        const uint64_t bits = __builtin_bit_cast(uint64_t, score);
        const uint64_t lo = (uint32_t)__builtin_amdgcn_ds_permute(to, (int)(uint32_t)bits);
        const uint64_t hi = (uint32_t)__builtin_amdgcn_ds_permute(to, (int)(uint32_t)(bits >> 32));
        lost |= li == p.k - 1 && list[TOP - 1] != 0 &&
                too_close(__builtin_bit_cast(double, hi << 32 | lo), score_of(list[TOP - 1] & ~MASK), route_margin(MASK));
      }
    }
    const bool used = li < p.k;
    if (!used) logit = -__builtin_inff();
    const uint64_t left = __ballot(lost);
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
    if (used && t0 + sub < p.tokens && (left >> lane0 & LANES) == 0) {
      p.weights[t * p.k + li] = (float)(w * p.scale);
      p.chosen[t * p.k + li] = mine;
    }
    if (left == 0) return;
    uint64_t* keys = s_key + wave * (p.experts + p.groups);
    for (int n = 0; n < TOKENS; ++n)
      if (t0 + n < p.tokens && (left >> (n * LPT) & LANES) != 0) route_token<E>(p, t0 + n, lane, keys, keys + p.experts);
  }
}

// Every token on 64-bit scores, one a wave: for lists longer than route_kernel's, and groups that its lanes cannot
// hold. Bound by the k rounds of a maximum over the wave: 16384 tokens, 8 of 256 experts 44 us, 4 of 8 groups too 64.
template <class E>
__global__ void __launch_bounds__(256) route_exact_kernel(RouteParams p) {
  extern __shared__ uint64_t s_key[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t* keys = s_key + wave * (p.experts + p.groups);
  const int t = (int)blockIdx.x * 4 + wave;
  if (t < p.tokens) route_token<E>(p, t, lane, keys, keys + p.experts);
}

// Gradient of the logits through the chosen scores.  64 / LPT tokens a wave; a lane of a token's first k holds a chosen
// expert. Where the gradient is not dense it is k numbers among zeros, put together in LDS and stored in whole lines.
// 16384 x 256 fp32 6.4 us, 2.6 TB/s written: bound by a launch and the chain of its steps (chosen, their logits, the
// exponential, LDS, stores), with vector instructions in 4 tenths of the busy cycles.  The dense one by 64-bit
// exponentials, 4097 x 896 bf16 9.6 us, 7 tenths.
template <class E, int LPT, int PER>
__global__ void __launch_bounds__(256) route_backward_kernel(RouteParams p) {
  constexpr int TOKENS = 64 / LPT;
  __shared__ __attribute__((aligned(16))) float s_row[4][TOKENS][LPT * PER];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int li = lane & (LPT - 1), sub = lane / LPT;
  const bool dense = !p.sigmoid && !p.normalize;
  float* row = s_row[wave][sub];
  const int t0 = ((int)blockIdx.x * 4 + wave) * TOKENS;
  if (t0 < p.tokens) {
    const int64_t t = min(t0 + sub, p.tokens - 1);
    const typename E::raw* x = static_cast<const typename E::raw*>(p.logits) + t * p.ldl;
    const int e = li < p.k ? p.chosen[t * p.k + li] : -1;
    const bool used = e >= 0 && e < p.experts;
    const double dw = used ? (double)p.dweights[t * p.k + li] * p.scale : 0;
    const float logit = used ? to_float<E>(x[e]) : -__builtin_inff();
    double s;
    if (p.sigmoid) {
      // s = 1 / (1 + z) or, of negative logits, z / (1 + z); s (1 - s) of either, where 1 - s has no bits left past 37.
      const double z = used ? exp(-fabs((double)logit)) : 0, inverse = 1 / (1 + z), slope = z * inverse * inverse;
      s = logit < 0 ? z * inverse : used ? inverse : 0;
      if (p.normalize) {
        const double total = token_sum<LPT>(s), mean = token_sum<LPT>(s * dw);
        s = total == 0 ? 0 : (dw - mean / total) * (slope / total);  // dw over a tiny total may be past the largest number
      } else {
        s = dw * slope;
      }
    } else if (dense) {
      double all[PER], total = 0;
      float v[PER], top = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        v[i] = to_float<E>(x[min(li + i * LPT, p.experts - 1)]);  // no branch around a load
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        v[i] = li + i * LPT < p.experts ? v[i] : -__builtin_inff();
        top = fmaxf(top, v[i]);
      }
      const float base = softmax_base(token_max<LPT>(top));
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        all[i] = exp((double)v[i] - base);
        total += all[i];
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
      total = token_sum<LPT>(total);
      const double inverse = total == 0 ? 0 : 1 / total;
      s = used ? exp((double)logit - base) * inverse : 0;
      const double mean = token_sum<LPT>(s * dw);
      s *= dw - mean;  // a small difference of large terms where s is close to 1
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
    if (used) row[e] = (float)s;  // in place of a dense gradient's part without dw
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    // The rows of the wave's tokens one after the other, 16 bytes a lane where they allow it.
    constexpr int N = 16 / sizeof(typename E::raw);
    const bool vec = p.experts % N == 0 && (reinterpret_cast<uintptr_t>(p.dlogits) & 15) == 0;
    for (int n = 0; n < TOKENS; ++n) {
      if (t0 + n >= p.tokens) break;
      typename E::raw* dx = static_cast<typename E::raw*>(p.dlogits) + (int64_t)(t0 + n) * p.experts;
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
  }
}

struct SortParams {
  const int32_t* experts;  // [n]
  int32_t* offs;           // [count]
  int32_t* slots;          // [n]
  int32_t* places;         // [n]
  int32_t* counts;         // workspace [blocks][count]
  int32_t n, first, count, chunk;  // chunk: entries of a workgroup, a multiple of 1024
};

// 64 N entries from `begin` on, one a lane each time, -1 for those that are none of the call's.
template <int N>
__device__ __forceinline__ void load_entries(const SortParams& p, int64_t begin, int (&e)[N]) {
  const int lane = threadIdx.x & 63;
  int raw[N];
#pragma unroll
  for (int i = 0; i < N; ++i)  // no branch around a load, but no load where there is no entry at all
    raw[i] = p.n > 0 ? p.experts[min(begin + i * 64 + lane, (int64_t)p.n - 1)] : 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t local = (int64_t)raw[i] - p.first;
    e[i] = begin + i * 64 + lane < p.n && local >= 0 && local < p.count ? (int)local : -1;
  }
}
template <int N>
__device__ __forceinline__ void count_entries(const int (&e)[N], int32_t* counts) {
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (e[i] >= 0) atomicAdd(&counts[e[i]], 1);
}
// An entry's place is its expert's next one in `next` plus the entries of its expert on lower lanes, found by matching
// the experts' bits across the lanes.
template <int N>
__device__ __forceinline__ void place_entries(const SortParams& p, int64_t begin, const int (&entries)[N], int32_t* next) {
  const int lane = threadIdx.x & 63;
  const int bits = p.count > 1 ? 32 - __builtin_clz((unsigned)(p.count - 1)) : 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t from = begin + i * 64 + lane;
    const int e = entries[i];
    uint64_t same = __ballot(e >= 0);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? set : ~set;
    }
    int base = 0;
    const int leader = e >= 0 ? __builtin_ctzll(same) : lane;
    if (e >= 0 && lane == leader) base = atomicAdd(&next[e], __builtin_popcountll(same));
    base = __shfl(base, leader);
    const int place = e >= 0 ? base + __builtin_popcountll(same & ((1ull << lane) - 1)) : -1;
    if (from < p.n) p.places[from] = place;
    if (place >= 0) p.slots[place] = (int32_t)from;
  }
}

// Exclusive sums over the workgroup's threads; `sums` holds one number a wave.  Every thread calls it.
template <int WAVES>
__device__ __forceinline__ int exclusive_sum(int x, int32_t* sums, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int sum = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int below = __shfl_up(sum, d);
    sum += lane >= d ? below : 0;
  }
  if (lane == 63) sums[wave] = sum;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const int n = sums[w];
    before += w < wave ? n : 0;
    all += n;
  }
  return before + sum - x;
}

// All of up to 1024 N entries in one workgroup of 16 waves: load, count, sum, place.  Counts are sums of integers and
// every order is that of the entries, so the result is the same at every call.  Bound by its steps' latencies: 512
// entries 3.4 us, 7108 10.2.
template <int N>
__global__ void __launch_bounds__(1024) sort_whole_kernel(SortParams p) {
  extern __shared__ int32_t s_next[];  // [16][count]
  __shared__ int32_t s_sums[16];
  const int wave = threadIdx.x >> 6;
  int entries[N];
  load_entries(p, wave * 64 * N, entries);
  for (int e = threadIdx.x; e < 16 * p.count; e += 1024) s_next[e] = 0;
  __syncthreads();
  int32_t* own = s_next + wave * p.count;
  count_entries(entries, own);
  __syncthreads();
  const int e = threadIdx.x;  // at most 1024 experts
  int counts[16], total = 0, used;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    counts[w] = e < p.count ? s_next[w * p.count + e] : 0;
    total += counts[w];
  }
  int at = exclusive_sum<16>(total, s_sums, used);
  if (e < p.count) {
    p.offs[e] = at + total;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      s_next[w * p.count + e] = at;
      at += counts[w];
    }
  }
  __syncthreads();
  place_entries(p, wave * 64 * N, entries, own);
  for (int i = used + threadIdx.x; i < p.n; i += 1024) p.slots[i] = -1;  // rows behind the last expert's
}

// How often each expert occurs in a workgroup's chunk.  32768 entries 4.8 us, a launch and two latencies.
__global__ void __launch_bounds__(256) sort_count_kernel(SortParams p) {
  __shared__ int32_t s_count[kSortExperts];
  for (int e = threadIdx.x; e < p.count; e += 256) s_count[e] = 0;
  __syncthreads();
  const int64_t begin = (int64_t)blockIdx.x * p.chunk + (threadIdx.x >> 6) * (p.chunk / 4);
  for (int i = 0; i < p.chunk / 4; i += 256) {
    int entries[4];
    load_entries(p, begin + i, entries);
    count_entries(entries, s_count);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.count; e += 256) p.counts[(int64_t)blockIdx.x * p.count + e] = s_count[e];
}

// Places of a workgroup's chunk: behind the smaller experts, the earlier workgroups and waves, and the wave's own
// earlier entries.  Each workgroup sums the counts of all for itself: reading them is cheaper than another launch.
// 32768 entries of 256 experts 7.9 us, bound by the latencies of reading entries, counts and entries again.
__global__ void __launch_bounds__(256) sort_place_kernel(SortParams p) {
  __shared__ int32_t s_next[4][kSortExperts];
  __shared__ int32_t s_total[kSortExperts], s_sums[4];
  const int wave = threadIdx.x >> 6;
  const int64_t begin = (int64_t)blockIdx.x * p.chunk;
  const int span = p.chunk / 4, blocks = (int)gridDim.x, block = (int)blockIdx.x;
  for (int e = threadIdx.x; e < 4 * kSortExperts; e += 256) (&s_next[0][0])[e] = 0;
  __syncthreads();
  int entries[4];
  for (int i = 0; i < span; i += 256) {
    load_entries(p, begin + wave * span + i, entries);
    count_entries(entries, s_next[wave]);
  }
  int before[kSortExperts / 256];
#pragma unroll
  for (int i = 0; i < kSortExperts / 256; ++i) {
    const int e = threadIdx.x + 256 * i;
    if (e >= p.count) break;
    int total = 0, earlier = 0;
    for (int b0 = 0; b0 < blocks; b0 += 16) {  // 16 counts on their way at a time
      int n[16];
#pragma unroll
      for (int b = 0; b < 16; ++b) n[b] = p.counts[(int64_t)min(b0 + b, blocks - 1) * p.count + e];
#pragma unroll
      for (int b = 0; b < 16; ++b) {
        total += b0 + b < blocks ? n[b] : 0;
        earlier += b0 + b < block ? n[b] : 0;
      }
    }
    s_total[e] = total;
    before[i] = earlier;
  }
  __syncthreads();
  int sum = 0, used;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = threadIdx.x * 4 + i;
    sum += e < p.count ? s_total[e] : 0;
  }
  int at = exclusive_sum<4>(sum, s_sums, used);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = threadIdx.x * 4 + i;
    if (e >= p.count) break;
    const int total = s_total[e];
    s_total[e] = at;  // where the expert starts
    at += total;
    if (block == 0) p.offs[e] = at;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSortExperts / 256; ++i) {
    const int e = threadIdx.x + 256 * i;
    if (e >= p.count) break;
    int next = s_total[e] + before[i];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int n = s_next[w][e];
      s_next[w][e] = next;
      next += n;
    }
  }
  __syncthreads();
  for (int i = 0; i < span; i += 256) {
    load_entries(p, begin + wave * span + i, entries);
    place_entries(p, begin + wave * span + i, entries, s_next[wave]);
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

// Sorted rows are read and written once by a call.  NT: they are too many to stay in the caches for the next one, and
// go past them (non-temporal), which leaves those to the tokens.
template <bool NT, class U>
__device__ __forceinline__ U load_row(const char* from) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const U*>(from));
  else return *reinterpret_cast<const U*>(from);
}
template <bool NT, class U>
__device__ __forceinline__ void store_row(char* to, U u) {
  if constexpr (NT) __builtin_nontemporal_store(u, reinterpret_cast<U*>(to));
  else *reinterpret_cast<U*>(to) = u;
}

// Rows that no token went to are zeros.
template <class U>
__device__ __forceinline__ void clear_rows(const RowsParams& p, int block, int blocks) {
  const int used = min(max(*p.end, 0), p.rows);
  for (int64_t r = used + block; r < p.rows; r += blocks)
    for (int64_t c = threadIdx.x * sizeof(U); c < p.width; c += 256 * sizeof(U))
      *reinterpret_cast<U*>(p.to + r * p.ld_to + c) = U{};
}

constexpr int kClearBlocks = 256;

// A token's places (and weights), one a lane; at(j) is slot j's, -1 where no row of the call belongs to it.
struct Places {
  int place;
  float weight;
  __device__ __forceinline__ void load(const RowsParams& p, int64_t t, int j0) {
    const int j = j0 + (int)(threadIdx.x & 63);
    const int64_t slot = t * p.k + min(j, p.k - 1);
    const int at = p.places[slot];
    weight = p.weights ? p.weights[slot] : 1.0f;
    place = at >= 0 && at < p.rows ? at : -1;
  }
  __device__ __forceinline__ int at(int j) const { return __builtin_amdgcn_readlane(place, j); }
  __device__ __forceinline__ float weight_at(int j) const {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), j));
  }
};

// A wave copies up to SPAN x 64 units of one token to all its places: a token is read once.  Bound by HBM's writes:
// 4096 tokens of 14336 bytes to 8 rows each 88 to 95 us, 5.6 to 6.0 TB/s read and written; 64 tokens of 4096 bytes 4.0
// us, launch and latency.
template <class U, bool NT>
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
    for (int j0 = 0; j0 < p.k; j0 += 64) {
      Places places;
      places.load(p, t, j0);
      for (int j = 0; j < min(p.k - j0, 64); ++j) {
        const int place = places.at(j);
        if (place < 0) continue;
        char* to = p.to + (int64_t)place * p.ld_to;
#pragma unroll
        for (int u = 0; u < SPAN; ++u) {
          const int64_t c = c0 + u * 64 * sizeof(U);
          if (c < p.width) store_row<NT>(to + c, v[u]);
        }
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

// A wave sums one span of a token's rows in the order of its slots, in fp32, and rounds once.  Four rows are on their
// way at a time.  Bound by HBM's reads: 4096 tokens of 14336 bytes from 8 rows each 88 to 91 us, 5.8 to 6.0 TB/s read
// and written.
template <class E, class U, bool NT>
__global__ void __launch_bounds__(256) combine_rows_kernel(RowsParams p) {
  using Q = Unit<E, U>;
  constexpr int SPAN = 2, AHEAD = 4;
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * 4;
  for (int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); item < p.tokens * p.spans; item += waves) {
    const int64_t t = item / p.spans;
    const int64_t c0 = ((item - t * p.spans) * SPAN * 64 + lane) * (int64_t)sizeof(U);
    float sum[SPAN][Q::N] = {};
    for (int j0 = 0; j0 < p.k; j0 += 64) {
      Places places;
      places.load(p, t, j0);
      const int count = min(p.k - j0, 64);
      for (int j = 0; j < count; j += AHEAD) {
        U v[AHEAD][SPAN] = {};
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
          const int place = places.at(min(j + a, count - 1));
          if (j + a >= count || place < 0) continue;
          const char* from = p.from + (int64_t)place * p.ld_from;
#pragma unroll
          for (int u = 0; u < SPAN; ++u) {
            const int64_t c = c0 + u * 64 * sizeof(U);
            if (c < p.width) v[a][u] = load_row<NT, U>(from + c);
          }
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
          if (j + a >= count || places.at(min(j + a, count - 1)) < 0) continue;
          const float w = places.weight_at(j + a);
#pragma unroll
          for (int u = 0; u < SPAN; ++u) {
            float f[Q::N];
            Q::widen(v[a][u], f);
#pragma unroll
            for (int i = 0; i < Q::N; ++i) sum[u][i] += w * f[i];
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < SPAN; ++u) {
      const int64_t c = c0 + u * 64 * sizeof(U);
      if (c < p.width) *reinterpret_cast<U*>(p.to + t * p.ld_to + c) = Q::narrow(sum[u]);
    }
  }
}

// One routed row a wave: dy = w dout and dw = <dout, y>, the product's sum over its lanes in one fixed order. Bound by
// HBM: 32768 rows of 14336 bytes, dy and dw, 190 us, 5.3 TB/s read and written, what a large copy reaches (4.85) and
// more.
template <class E, class U, bool NT>
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
          Q::widen(load_row<NT, U>(p.from + (int64_t)place * p.ld_from + c), y);
#pragma unroll
          for (int i = 0; i < Q::N; ++i) dot += d[i] * y[i];
        }
        if (p.to) {
#pragma unroll
          for (int i = 0; i < Q::N; ++i) d[i] *= w;
          store_row<NT>(p.to + (int64_t)place * p.ld_to + c, Q::narrow(d));
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
