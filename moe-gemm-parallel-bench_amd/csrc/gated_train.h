// Training form of the packed Gate+Up block over expert-sorted rows (gfx950): forward and backward.
//
//   forward:   [g | u] = x W_e,  h = silu(g) u                           (x [rows, H], W_e [H, 2F])
//   backward:  s = sigmoid(g),  dg = dh u s (1 + g (1 - s)),  du = dh g s,  dP = [dg | du]
//              dx = dP W_e^T,  dW_e = x_e^T dP_e
//
// Four launches: the forward product with h and [g | u] written by its epilogue, the elementwise dP, and
// the two products of the backward pass.  [g | u] is kept in fp32: rounded to 16 bits it would put two more
// roundings under every gradient, and recomputing it costs a third product (0.96 TFLOP, about 0.8 ms,
// against 0.27 GB written and read for 32 experts, 16384 rows, H 7168, F 2048).  dP is rounded to the
// operand type once, as the matrix cores take it: kept wider, as two 16-bit parts, it would double both products of
// the backward pass.  The rounding takes dx and dW from 0.0017 to 0.0024 of their norm off the 64-bit gradients in
// bf16, from 0.00021 to 0.00029 in fp16 (the lower figures are those of the outputs' own rounding).
//
// The products run on the LDS-DMA tiles (gemm_fast.h, gemm_pingpong.h): row-major operands forward,
// K-contiguous weights (kBT) for dx, the M-contiguous view of x (kAT) for dW, whose K is the expert's
// row count, read from the offsets on the device.  Rows are grouped as in MODE_OFFSETS; rows past the last
// group get h = 0 and dx = 0, an expert without rows dW = 0.
//
// 32 experts, 16384 rows, H 7168, F 2048, bf16, each product 0.96 TFLOP: forward 0.90 to 1.07 ms by card (0.03 less where
// the fp32 pairs are not kept), dX 0.90, dW 1.01, dP 0.079 (6.0 TB/s read and written).  The matrix instructions are busy half the time.  With
// uneven experts a sixth to a fifth of the row tiles' rows is padding, and workgroups that share weights drift apart: the
// forward pass fetches 4.0 GB where even experts fetch 2.3.  dW writes 1.9 GB, and each of its tiles (K is an
// expert's 512 rows) takes 18 us of which 4 are its epilogue and the next tile's start.
#pragma once

#include "fp8_gemm.h"
#include "gemm_pingpong.h"

namespace moegemm {

struct GatedParams {
  const void* x;      // [rows, h] (sx), or dP for dx
  const void* w;      // [groups, h, 2 f] (swg between groups, swh between rows)
  void* out;          // h [rows, f], dx [rows, h] or dW [groups, h, 2 f]
  float* saved;       // [rows, 2 f] gate | up, or null: not kept
  const void* dp;     // dW: dP [rows, 2 f]
  const int32_t* offs;
  int64_t sx, swg, swh, so, sog, sdp;  // element strides; so: row pitch of out, sog: dW's group stride
  int32_t groups, rows, h, f;  // groups: of this launch, [first, first + groups) of the call's
  int32_t long_k;     // dW: an expert's rows may span 2 GiB: K runs in segments
  int32_t first = 0;
  int32_t round = 0;   // the launch's first round of tiles
  int32_t closes = 1;  // the launch that clears what no tile writes past the last group
};

// Sums of one tile, as the tiles' run_tile forms them (FastTile::run_tile, PingPongTile::group_tile), with
// the epilogue left to `finish(acc, wave_m, wave_n)`, which every wave calls once its copies have landed.
template <class T>
struct TileSums {
  using acc_t = typename T::acc_t;
  static constexpr int FM = T::FM, FN = T::FN, ACC = T::ACC, KK = T::KK, BK = T::BK, STAGES = T::STAGES;
  static constexpr int XMIN = T::XMIN, NW = T::NW, WN = T::WN;

  __device__ static __forceinline__ void clear(acc_t (&acc)[FM][FN]) {
#pragma unroll
    for (int fm = 0; fm < FM; ++fm)
#pragma unroll
      for (int fn = 0; fn < FN; ++fn) acc[fm][fn] = acc_t{};
  }

  // K in segments of at most `segment` (a multiple of BK): one segment except where an operand's K
  // rows would span more than a buffer resource.  `at` moves the descriptor to a segment.
  template <bool SECOND, class At, class Finish>
  __device__ static __forceinline__ void ping_pong(const ProblemDesc& pd, int m0, int n0, int segment, char* smem,
                                                   At&& at, Finish&& finish) {
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int wave_m = wave / WN, wave_n = wave % WN;
    acc_t acc[FM][FN];
    clear(acc);
    int k0 = 0;
    do {
      const ProblemDesc part = at(pd, k0, segment);
      typename T::Dma d;
      T::setup_dma(d, part, m0, n0, smem);
#pragma unroll
      for (int s = 0; s < STAGES; ++s) T::template issue_stage<0>(d, s, s * BK);
      wait_vmcnt<(STAGES - 1) * XMIN>();
      phase_barrier();
      if constexpr (SECOND) phase_barrier();
      i16x8_t af[KK][FM], bf[KK][FN];
      const int kt_count = (part.k + BK - 1) / BK;
      for (int kt = 0; kt < kt_count; ++kt) {
        const char* cur = smem + (kt % STAGES) * T::STAGE_BYTES;
        if (kt >= 1) T::template issue_stage<0>(d, (kt - 1) % STAGES, (kt - 1 + STAGES) * BK);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          T::load_frags(af[kk], bf[kk], cur, cur + T::A_BYTES, kk, wave_m, wave_n, pd.swiglu != 0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if constexpr (SECOND) wait_vmcnt<(STAGES - 2) * XMIN>();
        phase_barrier();
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) T::template mfma_rows<0, FM>(acc, af[kk], bf[kk]);
        if constexpr (!SECOND) wait_vmcnt<(STAGES - 2) * XMIN>();
        phase_barrier();
      }
      wait_vmcnt<0>();
      k0 += segment;
      if (k0 < pd.k && !SECOND) phase_barrier();  // the groups are aligned again for the next segment
    } while (k0 < pd.k);
    finish(acc, wave_m, wave_n);
    if constexpr (!SECOND) phase_barrier();
  }

  template <class At, class Finish>
  __device__ static __forceinline__ void run(const ProblemDesc& pd, int m0, int n0, int segment, char* smem, At&& at,
                                             Finish&& finish) {
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if constexpr (std::is_base_of<PingPongTile<typename T::Element, BK, STAGES, T::LAY>, T>::value) {
      if (wave >= NW / 2)
        ping_pong<true>(pd, m0, n0, segment, smem, at, finish);
      else
        ping_pong<false>(pd, m0, n0, segment, smem, at, finish);
    } else {
      const int wave_m = wave / WN, wave_n = wave % WN;
      constexpr int HALF = FM / 2 > 0 ? FM / 2 : 1;
      acc_t acc[FM][FN];
      clear(acc);
      int k0 = 0;
      do {
        const ProblemDesc part = at(pd, k0, segment);
        typename T::Dma d;
        T::setup_dma(d, part, m0, n0, smem);
#pragma unroll
        for (int s = 0; s < STAGES; ++s) T::template issue_stage<0>(d, s, s * BK);
        wait_vmcnt<(STAGES - 1) * XMIN>();
        compiler_fence();
        __builtin_amdgcn_s_barrier();
        compiler_fence();
        i16x8_t af[2][FM], bf[2][FN];
        T::load_frags(af[0], bf[0], smem, smem + T::A_BYTES, 0, wave_m, wave_n, pd.swiglu != 0);
        const int kt_count = (part.k + BK - 1) / BK;
        for (int kt = 0; kt < kt_count; ++kt) {
          const char* cur = smem + (kt % STAGES) * T::STAGE_BYTES;
          const char* nxt = smem + ((kt + 1) % STAGES) * T::STAGE_BYTES;
#pragma unroll
          for (int kk = 0; kk < KK - 1; ++kk) {
            T::load_frags(af[(kk + 1) & 1], bf[(kk + 1) & 1], cur, cur + T::A_BYTES, kk + 1, wave_m, wave_n,
                          pd.swiglu != 0);
            T::template mfma_rows<0, FM>(acc, af[kk & 1], bf[kk & 1]);
            T::template interleave<FM * FN, T::FRAG_READS, 0>();
          }
          constexpr int L = (KK - 1) & 1;
          T::template mfma_rows<0, HALF>(acc, af[L], bf[L]);
          wait_vmcnt<(STAGES - 2) * XMIN>();
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          compiler_fence();
          __builtin_amdgcn_s_barrier();
          compiler_fence();
          T::template issue_stage<0>(d, kt % STAGES, (kt + STAGES) * BK);
          T::load_frags(af[0], bf[0], nxt, nxt + T::A_BYTES, 0, wave_m, wave_n, pd.swiglu != 0);
          T::template mfma_rows<HALF, FM>(acc, af[L], bf[L]);
          T::template interleave<(FM - HALF) * FN, T::FRAG_READS, T::QA + T::QB>();
        }
        wait_vmcnt<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        compiler_fence();
        __builtin_amdgcn_s_barrier();
        compiler_fence();
        k0 += segment;
      } while (k0 < pd.k);
      finish(acc, wave_m, wave_n);
    }
  }
};

// T::load_frags of the first half of a wave's rows.
template <class T>
__device__ __forceinline__ void load_half(i16x8_t (&af)[T::FM], i16x8_t (&bf)[T::FN], const char* stage, int kk, int wave_m,
                                          int wave_n, bool swiglu) {
#pragma unroll
  for (int fm = 0; fm < T::FM / 2; ++fm) {
    if constexpr (T::AT) af[fm] = T::frag_transposed(stage, T::CA, wave_m * T::WTM + fm * T::MI, kk);
    else af[fm] = T::frag_rows(stage, T::CA, wave_m * T::WTM + fm * T::MI, kk);
  }
#pragma unroll
  for (int fn = 0; fn < T::FN; ++fn) {
    const char* b = stage + T::A_BYTES;
    if constexpr (T::BT) bf[fn] = T::frag_rows(b, T::CB, wave_n * T::WTN + fn * T::MI, kk);
    else bf[fn] = T::frag_transposed(b, T::CB, T::b_frag_col(fn, wave_n, swiglu), kk);
  }
}

// Cross-tile chaining of the ping-pong tile (see PingPongTile::run_tile_chained) with an epilogue of the caller's.
// A tile's last three refills copy the next tile's slices 0 to 2; then the outputs leave in exactly Finish::STORES vector
// stores per wave, and slice 3 of the next tile follows.  A wave's vector memory operations complete in issue
// order, so the next tile waits for its slices by counting what is younger, stores included, and never for the stores
// before it needs slice 3.  `finish.chained(acc, pd, m0, n0, wave_m, wave_n, buffer)` may stage through the wave's
// slots of the last slice's buffer; `finish.last(...)` ends a tile without a successor.
struct ChainState {
  int rot;
  bool prefetched;
};

// The last row tile of a group of rows is rarely full: ROWS of the wave's FM row fragments (all, half, none) are
// loaded and multiplied, the others' outputs lie past the rows.
template <class T, bool SECOND, int ROWS, class Finish>
__device__ __forceinline__ void chained_tile(const ProblemDesc& pd, int m0, int n0, const ProblemDesc& next, int m1,
                                             int n1, bool has_next, char* smem, ChainState& ch, Finish&& finish) {
  constexpr int FM = T::FM, FN = T::FN, KK = T::KK, BK = T::BK, STAGES = T::STAGES, XMIN = T::XMIN;
  using F = typename std::remove_reference<Finish>::type;
  static_assert(STAGES == 4 && 3 * XMIN + F::STORES < 64, "outstanding operations must fit the 6-bit vmcnt");
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wave_m = wave / T::WN, wave_n = wave % T::WN;
  typename T::Dma d;
  T::setup_dma(d, pd, m0, n0, smem);
  typename T::acc_t acc[FM][FN];
  TileSums<T>::clear(acc);
  const bool pre = ch.prefetched;
  const int rot = pre ? ch.rot : 0;
  if (pre) {
    wait_vmcnt<3 * XMIN + F::STORES>();
  } else {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) T::template issue_stage<0>(d, s, s * BK);
    wait_vmcnt<(STAGES - 1) * XMIN>();
  }
  phase_barrier();
  if constexpr (SECOND) phase_barrier();
  const int kt_count = (pd.k + BK - 1) / BK;
  const bool chain = has_next && kt_count >= STAGES;
  i16x8_t af[KK][FM], bf[KK][FN];
  // ISSUE: 0 none, 1 this tile's slice kt + 3 (zeros past K), 2 the next tile's once that index passes K.
  auto step = [&](int kt, auto issue, auto edge) {
    constexpr int ISSUE = decltype(issue)::value;
    constexpr bool EDGE = decltype(edge)::value;
    const char* cur = smem + ((kt + rot) & (STAGES - 1)) * T::STAGE_BYTES;
    const int buffer = (kt - 1 + rot) & (STAGES - 1), s = kt - 1 + STAGES;
    if constexpr (ISSUE == 1) {
      T::template issue_stage<0>(d, buffer, s * BK);
    } else if constexpr (ISSUE == 2) {
      if (chain && s >= kt_count) {
        typename T::Dma dn;
        T::setup_dma(dn, next, m1, n1, smem);
        T::template issue_stage<0>(dn, buffer, (s - kt_count) * BK);
      } else {
        T::template issue_stage<0>(d, buffer, s * BK);
      }
    }
    if constexpr (ROWS == FM) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        T::load_frags(af[kk], bf[kk], cur, cur + T::A_BYTES, kk, wave_m, wave_n, pd.swiglu != 0);
    } else if constexpr (ROWS > 0) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) load_half<T>(af[kk], bf[kk], cur, kk, wave_m, wave_n, pd.swiglu != 0);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    auto wait_next = [&] {  // slice kt + 1 has landed
      if constexpr (EDGE) {
        if (!chain || kt + 1 < kt_count) {
          if (pre && kt < 2) wait_vmcnt<(STAGES - 2) * XMIN + F::STORES>();
          else wait_vmcnt<(STAGES - 2) * XMIN>();
        }
      } else {
        wait_vmcnt<(STAGES - 2) * XMIN>();
      }
    };
    if constexpr (SECOND) wait_next();
    phase_barrier();
    if constexpr (ROWS == FM) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) T::template mfma_rows<0, FM>(acc, af[kk], bf[kk]);
    } else if constexpr (ROWS > 0) {
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) T::template mfma_rows<0, ROWS>(acc, af[kk], bf[kk]);
    }
    if constexpr (!SECOND) wait_next();
    phase_barrier();
  };
  using none = std::integral_constant<int, 0>;
  using own = std::integral_constant<int, 1>;
  using either = std::integral_constant<int, 2>;
  step(0, none{}, std::true_type{});
  int kt = 1;
  for (; kt < 2 && kt < kt_count; ++kt) step(kt, either{}, std::true_type{});
  for (; kt + STAGES - 1 < kt_count; ++kt) step(kt, own{}, std::false_type{});
  for (; kt < kt_count; ++kt) step(kt, either{}, std::true_type{});
  if (chain) {
    const int last = (kt_count - 1 + rot) & (STAGES - 1);
    // The first group waits out the second's last products, so that both groups' epilogues run side by side (dW of 512
    // rows an expert 1 % faster than with one after the other).
    if constexpr (!SECOND) phase_barrier();
    finish.chained(acc, pd, m0, n0, wave_m, wave_n, last);
    typename T::Dma dn;
    T::setup_dma(dn, next, m1, n1, smem);
    T::template issue_stage<0>(dn, last, (STAGES - 1) * BK);
    ch.rot = (kt_count + rot) & (STAGES - 1);
    ch.prefetched = true;
  } else {
    wait_vmcnt<0>();
    finish.last(acc, pd, m0, n0, wave_m, wave_n);
    if constexpr (!SECOND) phase_barrier();
    ch.prefetched = false;
  }
}

// The tiles with their element type's name, which TileSums asks for.
template <class E, int BM, int BN, int BK, int WM, int WN, int S, int LAY>
struct GatedTile
    : std::conditional<BM == 256 && BN == 256, PingPongTile<E, BK, S, LAY>, FastTile<E, BM, BN, BK, WM, WN, S, LAY>>::type {
  using Element = E;
  static constexpr int PER_CU = 2 * (GatedTile::PREFIX_OFFSET + (int)(sizeof(TileTable) + sizeof(TileList))) <= 160 * 1024
                                    ? 2 : 1;
};

enum GatedProduct : int { GATED_FORWARD = 0, GATED_DX = 1, GATED_DW = 2 };

// h = silu(g) u and [g | u] of a tile, in a fixed number of buffer stores (out-of-range lanes are dropped): gate
// fragments and the up fragments FN / 2 further on.  A lane holds four consecutive columns of one row per register quad;
// 32x32 fragments go through the wave's slots of one stage in LDS, so that stores write 128 (fp32) and 64 bytes of a
// row at a time instead of 32 (16-byte chunk c of a row at c ^ row).  Non-temporal: the operands keep the L2 (8 experts, 4096
// rows, 4096 -> 2x1536: 127 us with ordinary stores, 100 so).
template <class T>
struct StoreGateUp {
  using E = typename T::Element;
  static constexpr int FRAGS = T::FM * (T::FN / 2);
  static constexpr int STORES = T::MI == 32 ? 10 * FRAGS : 3 * FRAGS;
  float* saved;  // the group's first row, or null
  int64_t f;
  char* smem;

  __device__ __forceinline__ void last(const typename T::acc_t (&acc)[T::FM][T::FN], const ProblemDesc& pd, int m0,
                                       int n0, int wave_m, int wave_n) const {
    chained(acc, pd, m0, n0, wave_m, wave_n, 0);
  }
  __device__ __forceinline__ void chained(const typename T::acc_t (&acc)[T::FM][T::FN], const ProblemDesc& pd, int m0,
                                          int n0, int wave_m, int wave_n, int stage) const {
    const int lane = lane_here();
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    constexpr int MI = T::MI;
    const int rows = min(T::BM, pd.m - m0), cols = (int)f - n0 / 2;
    const uint32_t pitch = (uint32_t)pd.scm * 2u, pitch32 = (uint32_t)f * 8u;
    float* keep = saved + (int64_t)m0 * 2 * f + n0 / 2;
    const int kept = (int)(saved ? kOutOfRange : 0);  // a resource of no bytes drops the stores, whose count stays
    const auto rh = __builtin_amdgcn_make_buffer_rsrc(pd.c + ((int64_t)m0 * pd.scm + n0 / 2) * 2, (short)0,
                                                      (int)kOutOfRange, (int)kBufferFlags);
    const auto rg = __builtin_amdgcn_make_buffer_rsrc(keep, (short)0, kept, (int)kBufferFlags);
    const auto ru = __builtin_amdgcn_make_buffer_rsrc(keep + f, (short)0, kept, (int)kBufferFlags);
#pragma unroll
    for (int fm = 0; fm < T::FM; ++fm)
#pragma unroll
      for (int fn = 0; fn < T::FN / 2; ++fn) {
        const int row0 = wave_m * T::WTM + fm * MI, n1 = wave_n * (T::WTN / 2) + fn * MI;
        f32x4_t v[2][T::ACC / 4];
        u32x2_t h[T::ACC / 4];
#pragma unroll
        for (int q = 0; q < T::ACC / 4; ++q) {
          f32x4_t x;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[0][q][i] = acc[fm][fn][q * 4 + i];
            v[1][q][i] = acc[fm][fn + T::FN / 2][q * 4 + i];
            x[i] = gated(v[0][q][i], v[1][q][i]);
          }
          h[q] = pack4<E>(x);
        }
        if constexpr (MI == 16) {
          const int row = row0 + lane % 16, n = n1 + (lane >> 4) * 4;
          const bool in = row < rows && n < cols;
          const uint32_t at = in ? (uint32_t)row * pitch32 + (uint32_t)n * 4u : kOutOfRange;
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v[0][0]), rg, at, 0, 0);
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v[1][0]), ru, at, 0, 0);
          __builtin_amdgcn_raw_buffer_store_b64(h[0], rh, in ? (uint32_t)row * pitch + (uint32_t)n * 2u : kOutOfRange, 0, 0);
        } else {
          static_assert(MI == 16 || T::XMIN >= 4, "a 32 x 32 fp32 fragment takes four 1 KiB slots");
          auto slot = [&](int linear) {
            return smem + T::owned_slot(stage * T::XMIN + (linear >> 10), wave) + (linear & 1023);
          };
          const int r = lane & 31;
#pragma unroll
          for (int part = 0; part < 2; ++part) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<f32x4_t*>(slot(r * 128 + (((q * 2 + (lane >> 5)) ^ (r & 7)) << 4))) = v[part][q];
            compiler_fence();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int row = j * 8 + (lane >> 3), c = lane & 7;
              const u32x4_t x = *reinterpret_cast<const u32x4_t*>(slot(row * 128 + ((c ^ (row & 7)) << 4)));
              const bool in = row0 + row < rows && n1 + c * 4 < cols;
              const uint32_t at = (uint32_t)(row0 + row) * pitch32 + (uint32_t)(n1 + c * 4) * 4u;
              __builtin_amdgcn_raw_buffer_store_b128(x, part ? ru : rg, in ? at : kOutOfRange, 0, kNonTemporal);
            }
            compiler_fence();
          }
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<u32x2_t*>(slot(r * 64 + ((q ^ (r & 3)) << 4) + (lane >> 5) * 8)) = h[q];
          compiler_fence();
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int row = j * 16 + (lane >> 2), c = lane & 3;
            const u32x4_t x = *reinterpret_cast<const u32x4_t*>(slot(row * 64 + ((c ^ (row & 3)) << 4)));
            const bool in = row0 + row < rows && n1 + c * 8 < cols;
            __builtin_amdgcn_raw_buffer_store_b128(
                x, rh, in ? (uint32_t)(row0 + row) * pitch + (uint32_t)(n1 + c * 8) * 2u : kOutOfRange, 0, 0);
          }
          compiler_fence();
        }
      }
  }
};

// C of a plain product.
template <class T>
struct StorePlain {
  static constexpr int STORES = T::CHAIN_STORES;
  char* smem;
  __device__ __forceinline__ void last(const typename T::acc_t (&acc)[T::FM][T::FN], const ProblemDesc& pd, int m0,
                                       int n0, int wave_m, int wave_n) const {
    T::template store_tile<EPI_C>(acc, pd, m0, n0, wave_m, wave_n, smem);
  }
  __device__ __forceinline__ void chained(const typename T::acc_t (&acc)[T::FM][T::FN], const ProblemDesc& pd, int m0,
                                          int n0, int wave_m, int wave_n, int buffer) const {
    T::staged_store_counted(acc, pd, m0, n0, wave_m, wave_n, smem, buffer);
  }
};

// Zeros to rows [first, rows) of a [rows, width] 16-bit matrix (row pitch in elements, width and pitch
// multiples of 8, 16-byte aligned), every thread of the launch.
__device__ __forceinline__ void zero_rows(void* base, int64_t pitch, int width, int64_t first, int64_t rows) {
  const int64_t chunks = (rows - first) * (width / 8);
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = first + i / (width / 8), c = i % (width / 8);
    *reinterpret_cast<u32x4_t*>(static_cast<char*>(base) + (row * pitch + c * 8) * 2) = u32x4_t{};
  }
}

// First row past the last group, in [0, rows].
__device__ __forceinline__ int rows_end(const GatedParams& p) {
  return p.offs ? min(max(p.offs[p.first + p.groups - 1], 0), p.rows) : p.rows;
}

constexpr int kWholeK = 1 << 30;  // no segments

// LDS of a workgroup: the tile's stages, then the tables.
template <class T>
constexpr int kGatedLds = T::PREFIX_OFFSET + (int)(sizeof(TileTable) + sizeof(TileList));

template <class T, int PRODUCT>
__global__ void __launch_bounds__(T::NT) gated_product_kernel(GatedParams p) {
  __shared__ __attribute__((aligned(16))) char smem[kGatedLds<T>];
  static_assert(kGatedLds<T> <= 160 * 1024, "LDS of one CU");
  TileTable& table = *reinterpret_cast<TileTable*>(smem + T::PREFIX_OFFSET);
  TileList& list = *reinterpret_cast<TileList*>(smem + T::PREFIX_OFFSET + sizeof(TileTable));
  const int n = PRODUCT == GATED_DX ? p.h : 2 * p.f;
  // dW: every expert with rows holds the same number of tiles.
  constexpr int ROWS_PER_TILE = PRODUCT == GATED_DW ? 1 << 30 : T::BM;
  const int n_tiles = (n + T::BN - 1) / T::BN, m_tiles = (p.h + T::BM - 1) / T::BM;
  const int per_row_tile = PRODUCT == GATED_DW ? m_tiles * n_tiles : n_tiles;
  const char* x = static_cast<const char*>(p.x);
  const char* w = static_cast<const char*>(p.w);
  char* out = static_cast<char*>(p.out);

  build_tile_table(table, p.offs, p.first, p.groups, p.rows, ROWS_PER_TILE, per_row_tile);

  auto describe = [&](int i, ProblemDesc& pd, int& m0, int& n0, float*& saved) {  // the list's i-th tile
    GroupTile g;
    if (!listed_tile(list, i, g)) return false;
    pd = ProblemDesc{};
    pd.splits = 1;
    pd.scn = 1;
    pd.scm = p.so;
    pd.n = n;
    if constexpr (PRODUCT == GATED_DW) {
      pd.a = x + (int64_t)g.row0 * p.sx * 2;
      pd.b = static_cast<const char*>(p.dp) + (int64_t)g.row0 * p.sdp * 2;
      pd.c = out + (int64_t)g.e * p.sog * 2;
      pd.m = p.h; pd.k = g.m;
      pd.sam = 1; pd.sak = p.sx; pd.sbk = p.sdp; pd.sbn = 1;
    } else {
      pd.a = x + (int64_t)g.row0 * p.sx * 2;
      pd.b = w + (int64_t)g.e * p.swg * 2;
      pd.c = out + (int64_t)g.row0 * p.so * 2;
      pd.m = g.m;
      pd.sam = p.sx; pd.sak = 1;
      if constexpr (PRODUCT == GATED_FORWARD) {
        pd.k = p.h;
        pd.sbk = p.swh; pd.sbn = 1;
        pd.swiglu = 1;
        saved = p.saved ? p.saved + (int64_t)g.row0 * 2 * p.f : nullptr;
      } else {
        pd.k = 2 * p.f;
        pd.sbk = 1; pd.sbn = p.swh;
      }
    }
    make_uniform(pd);
    m0 = g.tm * T::BM + g.part;
    n0 = g.tn * T::BN;
    return true;
  };
  constexpr bool PING_PONG = T::BM == 256 && T::BN == 256;
  auto finish = [&](float* saved) {
    if constexpr (PRODUCT == GATED_FORWARD) return StoreGateUp<T>{saved, p.f, smem};
    else return StorePlain<T>{smem};
  };

  // A short last round in parts: 4096 rows of 8 experts, H 4096, F 1536, dX 152 us whole, 142 in parts; 4001 of 16, H and
  // F 2880, 299 and 276; forward of 16384 uneven rows, 7168 -> 2x2048 (an eighth of a round left), 994 and 987.
  build_tile_list<PING_PONG && PRODUCT != GATED_DW ? T::BM : 0>(list, table, p.first, p.groups, p.round,
                                                                [&](GroupTile& tile, int local) {
    group_m_order(local, PRODUCT == GATED_DW ? m_tiles : (tile.m + T::BM - 1) / T::BM, n_tiles, 8, tile.tm, tile.tn);
  });
  ProblemDesc pd;
  int m0 = 0, n0 = 0, i = 0;
  float* saved = nullptr;
  bool more = describe(0, pd, m0, n0, saved);
  if (PING_PONG && !p.long_k) {
    if constexpr (PING_PONG) {
      ChainState ch{0, false};
      while (more) {
        ProblemDesc next;
        int m1 = 0, n1 = 0;
        float* saved_next = nullptr;
        more = describe(++i, next, m1, n1, saved_next);
        auto tile = [&](auto second, auto rows) {
          chained_tile<T, decltype(second)::value, decltype(rows)::value>(pd, m0, n0, next, m1, n1, more, smem, ch,
                                                                           finish(saved));
        };
        using all = std::integral_constant<int, T::FM>;
        using half = std::integral_constant<int, T::FM / 2>;
        const int rows = PRODUCT == GATED_DW ? T::BM : pd.m - m0;
        if (__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) >= T::NW / 2) {
          if (rows > T::BM / 2 + T::WTM / 2) tile(std::true_type{}, all{});
          else if (rows > T::BM / 2) tile(std::true_type{}, half{});
          else tile(std::true_type{}, std::integral_constant<int, 0>{});
        } else {
          if (rows > T::WTM / 2) tile(std::false_type{}, all{});
          else tile(std::false_type{}, half{});
        }
        pd = next;
        m0 = m1;
        n0 = n1;
        saved = saved_next;
      }
    }
  } else {
    while (more) {
      auto store = [&](const typename T::acc_t (&acc)[T::FM][T::FN], int wave_m, int wave_n) {
        finish(saved).last(acc, pd, m0, n0, wave_m, wave_n);
      };
      if (PRODUCT == GATED_DW && p.long_k) {
        const int64_t pitch = max(p.sx, p.sdp) * 2;
        const int segment = (int)(((int64_t)1 << 30) / pitch / T::BK) * T::BK;  // 2^30 bytes of rows at a time
        TileSums<T>::run(pd, m0, n0, segment, smem, [](const ProblemDesc& whole, int k0, int length) {
          ProblemDesc part = whole;
          part.a += (int64_t)k0 * whole.sak * 2;
          part.b += (int64_t)k0 * whole.sbk * 2;
          part.k = min(length, whole.k - k0);
          return part;
        }, store);
      } else {
        TileSums<T>::run(pd, m0, n0, kWholeK, smem, [](const ProblemDesc& whole, int, int) { return whole; }, store);
      }
      more = describe(++i, pd, m0, n0, saved);
    }
  }

  // What no tile writes: rows past the last group, gradients of experts without rows.  After the tiles, whose first
  // loads it would delay.
  if constexpr (PRODUCT == GATED_DW) {
    for (int first = 0; p.round == 0 && first < p.groups; first += 64) {
      const int e = first + (int)(threadIdx.x & 63);
      const bool none = e < p.groups && table.tiles[e] == (e ? table.tiles[e - 1] : 0);
      for (uint64_t empty = __builtin_amdgcn_ballot_w64(none); empty; empty &= empty - 1)
        zero_rows(out + (int64_t)(p.first + first + __builtin_ctzll(empty)) * p.sog * 2, p.so, n, 0, p.h);
    }
  } else if (p.closes) {
    zero_rows(out, p.so, PRODUCT == GATED_DX ? p.h : p.f, table.ends[p.groups - 1], p.rows);
  }
}

// dP = [dg | du] from dh and the saved [g | u], 8 columns of each half a thread; rows past the last group
// are not read by any product and stay unwritten.
template <class E>
__global__ void __launch_bounds__(256) gate_up_gradient_kernel(GatedParams p, const void* dh, int64_t sdh, void* dp) {
  const int chunks = p.f / 8;
  const int64_t total = (int64_t)rows_end(p) * chunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / chunks;
    const int col = (int)(i % chunks) * 8;
    const float* keep = p.saved + row * 2 * p.f + col;
    const f32x4_t* g4 = reinterpret_cast<const f32x4_t*>(keep);
    const f32x4_t* u4 = reinterpret_cast<const f32x4_t*>(keep + p.f);
    const u32x4_t raw = *reinterpret_cast<const u32x4_t*>(static_cast<const char*>(dh) + (row * sdh + col) * 2);
    u32x4_t dg, du;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const f32x4_t g = g4[half], u = u4[half];
      f32x4_t a, b;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t word = raw[half * 2 + j / 2];
        const uint16_t bits = (uint16_t)(j & 1 ? word >> 16 : word);
        float d;
        if constexpr (E::dtype == DT_BF16) d = __builtin_bit_cast(float, (uint32_t)bits << 16);
        else d = (float)__builtin_bit_cast(_Float16, bits);
        const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-g[j]));
        a[j] = d * u[j] * (s * (1.0f + g[j] * (1.0f - s)));
        b[j] = d * (g[j] * s);
      }
      const u32x2_t pa = pack4<E>(a), pb = pack4<E>(b);
      dg[half * 2] = pa[0]; dg[half * 2 + 1] = pa[1];
      du[half * 2] = pb[0]; du[half * 2 + 1] = pb[1];
    }
    char* to = static_cast<char*>(dp) + (row * 2 * p.f + col) * 2;
    *reinterpret_cast<u32x4_t*>(to) = dg;
    *reinterpret_cast<u32x4_t*>(to + (int64_t)p.f * 2) = du;
  }
}

typedef hipError_t (*GatedLaunchFn)(const GatedParams&, int grid, hipStream_t stream);
struct GatedVariant {
  int block_m, block_n, per_cu;  // per_cu: workgroups a CU holds (LDS and registers)
  int slice_ps, tile_ns, gbps;
  GatedLaunchFn launch;
};
template <class T, int PRODUCT>
hipError_t launch_gated(const GatedParams& p, int grid, hipStream_t stream) {
  hipLaunchKernelGGL((gated_product_kernel<T, PRODUCT>), dim3(grid), dim3(T::NT), 0, stream, p);
  return hipGetLastError();
}
template <class E>
hipError_t launch_gradient(const GatedParams& p, const void* dh, int64_t sdh, void* dp, int grid, hipStream_t stream) {
  hipLaunchKernelGGL((gate_up_gradient_kernel<E>), dim3(grid), dim3(256), 0, stream, p, dh, sdh, dp);
  return hipGetLastError();
}

// X(E, BM, BN, BK, WAVES_M, WAVES_N, STAGES, layout, product, ps, ns, gbps), largest tiles first; the last three are
// what the choice of a variant reckons with, measured on full chips: a round of one tile per workgroup takes ps
// picoseconds per element of K and ns nanoseconds besides, and weights that few rows share arrive at gbps.
#define MOEGEMM_MENU_GATED(X, E)                                   \
  X(E, 256, 256, 32, 2, 4, 4, 0, GATED_FORWARD, 26000, 5000, 5400) \
  X(E, 128, 256, 64, 2, 4, 3, 0, GATED_FORWARD, 16500, 4000, 5400) \
  X(E, 64, 128, 64, 2, 2, 4, 0, GATED_FORWARD, 6800, 2300, 4300)   \
  X(E, 16, 128, 128, 1, 4, 4, 0, GATED_FORWARD, 5500, 2000, 3800)
#define MOEGEMM_MENU_DX(X, E)                                 \
  X(E, 256, 256, 32, 2, 4, 4, 2, GATED_DX, 26000, 5000, 4500) \
  X(E, 128, 256, 64, 2, 4, 3, 2, GATED_DX, 16500, 4000, 4850) \
  X(E, 64, 64, 64, 2, 2, 4, 2, GATED_DX, 8200, 2300, 4850)    \
  X(E, 16, 64, 128, 1, 4, 4, 2, GATED_DX, 2600, 2000, 4100)
#define MOEGEMM_MENU_DW(X, E)                                 \
  X(E, 256, 256, 32, 2, 4, 4, 1, GATED_DW, 26000, 5000, 5400) \
  X(E, 128, 256, 64, 2, 4, 3, 1, GATED_DW, 16500, 4000, 5400) \
  X(E, 64, 64, 64, 2, 2, 4, 1, GATED_DW, 8200, 2300, 5400)
#define MOEGEMM_GATED_KERNEL(E, BM, BN, BK, WM, WN, S, LAY, PRODUCT, PS, NS, GBPS) \
  template __global__ void gated_product_kernel<GatedTile<E, BM, BN, BK, WM, WN, S, LAY>, PRODUCT>(GatedParams);
#define MOEGEMM_GATED_ENTRY(E, BM, BN, BK, WM, WN, S, LAY, PRODUCT, PS, NS, GBPS)           \
  GatedVariant{BM, BN, GatedTile<E, BM, BN, BK, WM, WN, S, LAY>::PER_CU, PS, NS, GBPS,      \
               &launch_gated<GatedTile<E, BM, BN, BK, WM, WN, S, LAY>, PRODUCT>},

// Per type (bf16, fp16): the variants of the three products, each list closed by a null launch.
struct GatedTable {
  const GatedVariant* products[3];
  hipError_t (*gradient)(const GatedParams&, const void*, int64_t, void*, int, hipStream_t);
};
extern const GatedTable kGatedBf16, kGatedF16;

}  // namespace moegemm
