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
// operand type once, as the matrix cores take it.
//
// The products run on the LDS-DMA tiles (gemm_fast.h, gemm_pingpong.h): row-major operands forward,
// K-contiguous weights (kBT) for dx, the M-contiguous view of x (kAT) for dW, whose K is the expert's
// row count, read from the offsets on the device.  Rows are grouped as in MODE_OFFSETS; rows past the last
// group get h = 0 and dx = 0, an expert without rows dW = 0.
#pragma once

#include "fp8_gemm.h"
#include "gemm_pingpong.h"

namespace moegemm {

struct GatedParams {
  const void* x;      // [rows, h] (sx), or dP for dx
  const void* w;      // [groups, h, 2 f] (swg between groups, swh between rows)
  void* out;          // h [rows, f], dx [rows, h] or dW [groups, h, 2 f]
  float* saved;       // [rows, 2 f] gate | up
  const void* dp;     // dW: dP [rows, 2 f]
  const int32_t* offs;
  int64_t sx, swg, swh, so, sog, sdp;  // element strides; so: row pitch of out, sog: dW's group stride
  int32_t groups, rows, h, f;
  int32_t long_k;     // dW: an expert's rows may span 2 GiB: K runs in segments
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

// The tiles with their element type's name, which TileSums asks for.
template <class E, int BM, int BN, int BK, int WM, int WN, int S, int LAY>
struct GatedTile
    : std::conditional<BM == 256 && BN == 256, PingPongTile<E, BK, S, LAY>, FastTile<E, BM, BN, BK, WM, WN, S, LAY>>::type {
  using Element = E;
};

enum GatedProduct : int { GATED_FORWARD = 0, GATED_DX = 1, GATED_DW = 2 };

// h = silu(g) u and [g | u] of a tile: gate fragments and the up fragments FN / 2 further on, four
// consecutive columns of one row per lane and register quad.
template <class T>
__device__ __forceinline__ void store_gate_up(const typename T::acc_t (&acc)[T::FM][T::FN], const ProblemDesc& pd,
                                              float* saved, int64_t f, int m0, int n0, int wave_m, int wave_n) {
  using E = typename T::Element;
  const int lane = threadIdx.x & 63;
  constexpr int MI = T::MI;
#pragma unroll
  for (int fm = 0; fm < T::FM; ++fm) {
    const int row = m0 + wave_m * T::WTM + fm * MI + (lane % MI);
    if (row >= pd.m) continue;
    char* out = pd.c + (int64_t)row * pd.scm * 2;
    float* keep = saved + (int64_t)row * 2 * f;
#pragma unroll
    for (int fn = 0; fn < T::FN / 2; ++fn)
#pragma unroll
      for (int q = 0; q < T::ACC / 4; ++q) {
        const int n = n0 / 2 + wave_n * (T::WTN / 2) + fn * MI + (MI == 32 ? q * 8 + (lane >> 5) * 4 : (lane >> 4) * 4);
        if (n >= f) continue;
        f32x4_t g, u, h;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          g[i] = acc[fm][fn][q * 4 + i];
          u[i] = acc[fm][fn + T::FN / 2][q * 4 + i];
          h[i] = gated(g[i], u[i]);
        }
        store4<E>(out + (int64_t)n * 2, h);
        *MOEGEMM_GLOBAL(f32x4_t, keep + n) = g;
        *MOEGEMM_GLOBAL(f32x4_t, keep + f + n) = u;
      }
  }
}

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
  return p.offs ? min(max(p.offs[p.groups - 1], 0), p.rows) : p.rows;
}

constexpr int kWholeK = 1 << 30;  // no segments

template <class T, int PRODUCT>
__global__ void __launch_bounds__(T::NT) gated_product_kernel(GatedParams p) {
  __shared__ __attribute__((aligned(16))) char smem[T::LDS_BYTES];
  const int grid = gridDim.x;
  int t = (int)blockIdx.x;
  if ((grid & 7) == 0) t = (t & 7) * (grid >> 3) + (t >> 3);  // eight contiguous runs a round, one per XCD
  const int n = PRODUCT == GATED_DX ? p.h : 2 * p.f;
  const int n_tiles = (n + T::BN - 1) / T::BN;
  const char* x = static_cast<const char*>(p.x);
  const char* w = static_cast<const char*>(p.w);
  char* out = static_cast<char*>(p.out);

  // What no tile writes: rows past the last group, gradients of experts without rows.
  if constexpr (PRODUCT == GATED_DW) {
    for (int first = 0; first < p.groups; first += 64) {
      const int e = first + (int)(threadIdx.x & 63);
      int m = 1;
      if (e < p.groups) group_rows(p.offs, p.rows, e, m);
      for (uint64_t empty = __builtin_amdgcn_ballot_w64(m == 0); empty; empty &= empty - 1)
        zero_rows(out + (int64_t)(first + __builtin_ctzll(empty)) * p.sog * 2, p.so, n, 0, p.h);
    }
  } else {
    zero_rows(out, p.so, PRODUCT == GATED_DX ? p.h : p.f, rows_end(p), p.rows);
  }

  auto whole = [](const ProblemDesc& pd, int, int) { return pd; };
  if constexpr (PRODUCT == GATED_DW) {
    // Every expert with rows holds the same number of tiles.
    const int m_tiles = (p.h + T::BM - 1) / T::BM;
    GroupTile g;
    for (; find_group_tile(p.offs, p.groups, p.rows, 1 << 30, m_tiles * n_tiles, t, g); t += grid) {
      int tm, tn;
      group_m_order(g.local, m_tiles, n_tiles, 8, tm, tn);
      ProblemDesc pd{};
      pd.a = x + (int64_t)g.row0 * p.sx * 2;
      pd.b = static_cast<const char*>(p.dp) + (int64_t)g.row0 * p.sdp * 2;
      pd.c = out + (int64_t)g.e * p.sog * 2;
      pd.m = p.h; pd.n = n; pd.k = g.m;
      pd.sam = 1; pd.sak = p.sx; pd.sbk = p.sdp; pd.sbn = 1; pd.scm = p.so; pd.scn = 1;
      pd.splits = 1;
      const int m0 = tm * T::BM, n0 = tn * T::BN;
      auto store = [&](const typename T::acc_t (&acc)[T::FM][T::FN], int wave_m, int wave_n) {
        T::template store_tile<EPI_C>(acc, pd, m0, n0, wave_m, wave_n, smem);
      };
      if (p.long_k) {
        // 2^30 bytes of rows at a time.
        const int64_t pitch = max(p.sx, p.sdp) * 2;
        const int segment = (int)(((int64_t)1 << 30) / pitch / T::BK) * T::BK;
        TileSums<T>::run(pd, m0, n0, segment, smem, [](const ProblemDesc& whole, int k0, int length) {
          ProblemDesc part = whole;
          part.a += (int64_t)k0 * whole.sak * 2;
          part.b += (int64_t)k0 * whole.sbk * 2;
          part.k = min(length, whole.k - k0);
          return part;
        }, store);
      } else {
        TileSums<T>::run(pd, m0, n0, kWholeK, smem, whole, store);
      }
    }
  } else {
    GroupTile g;
    for (; find_group_tile(p.offs, p.groups, p.rows, T::BM, n_tiles, t, g); t += grid) {
      int tm, tn;
      group_m_order(g.local, (g.m + T::BM - 1) / T::BM, n_tiles, 8, tm, tn);
      ProblemDesc pd{};
      pd.a = x + (int64_t)g.row0 * p.sx * 2;
      pd.b = w + (int64_t)g.e * p.swg * 2;
      pd.c = out + (int64_t)g.row0 * p.so * 2;
      pd.m = g.m; pd.n = n;
      pd.sam = p.sx; pd.sak = 1; pd.scm = p.so; pd.scn = 1;
      pd.splits = 1;
      const int m0 = tm * T::BM, n0 = tn * T::BN;
      if constexpr (PRODUCT == GATED_FORWARD) {
        pd.k = p.h;
        pd.sbk = p.swh; pd.sbn = 1;
        pd.swiglu = 1;
        TileSums<T>::run(pd, m0, n0, kWholeK, smem, whole,
                         [&](const typename T::acc_t (&acc)[T::FM][T::FN], int wave_m, int wave_n) {
                           store_gate_up<T>(acc, pd, p.saved + (int64_t)g.row0 * 2 * p.f, p.f, m0, n0, wave_m, wave_n);
                         });
      } else {
        pd.k = 2 * p.f;
        pd.sbk = 1; pd.sbn = p.swh;
        TileSums<T>::run(pd, m0, n0, kWholeK, smem, whole,
                         [&](const typename T::acc_t (&acc)[T::FM][T::FN], int wave_m, int wave_n) {
                           T::template store_tile<EPI_C>(acc, pd, m0, n0, wave_m, wave_n, smem);
                         });
      }
    }
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
  int block_m, block_n;
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

// X(E, BM, BN, BK, WAVES_M, WAVES_N, STAGES, layout, product), largest tiles first.
#define MOEGEMM_MENU_GATED(X, E)                                                        \
  X(E, 256, 256, 32, 2, 4, 4, 0, GATED_FORWARD) X(E, 128, 256, 64, 2, 4, 3, 0, GATED_FORWARD) \
  X(E, 64, 128, 64, 2, 2, 4, 0, GATED_FORWARD) X(E, 16, 128, 128, 1, 4, 4, 0, GATED_FORWARD)
#define MOEGEMM_MENU_DX(X, E)                                                           \
  X(E, 256, 256, 32, 2, 4, 4, 2, GATED_DX) X(E, 128, 256, 64, 2, 4, 3, 2, GATED_DX)     \
  X(E, 64, 64, 64, 2, 2, 4, 2, GATED_DX) X(E, 16, 64, 128, 1, 4, 4, 2, GATED_DX)
#define MOEGEMM_MENU_DW(X, E)                                                           \
  X(E, 256, 256, 32, 2, 4, 4, 1, GATED_DW) X(E, 128, 256, 64, 2, 4, 3, 1, GATED_DW)     \
  X(E, 64, 64, 64, 2, 2, 4, 1, GATED_DW)
#define MOEGEMM_GATED_KERNEL(E, BM, BN, BK, WM, WN, S, LAY, PRODUCT) \
  template __global__ void gated_product_kernel<GatedTile<E, BM, BN, BK, WM, WN, S, LAY>, PRODUCT>(GatedParams);
#define MOEGEMM_GATED_ENTRY(E, BM, BN, BK, WM, WN, S, LAY, PRODUCT) \
  GatedVariant{BM, BN, &launch_gated<GatedTile<E, BM, BN, BK, WM, WN, S, LAY>, PRODUCT>},

// Per type (bf16, fp16): the variants of the three products, each list closed by a null launch.
struct GatedTable {
  const GatedVariant* products[3];
  hipError_t (*gradient)(const GatedParams&, const void*, int64_t, void*, int, hipStream_t);
};
extern const GatedTable kGatedBf16, kGatedF16;

}  // namespace moegemm
