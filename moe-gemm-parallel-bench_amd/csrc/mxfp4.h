// Products of 16-bit rows with 4-bit weights (MXFP4), and the format's conversions (gfx950).
//
//   C[m, n] = sum_k a[m, k] v[n, k] 2^(s[n, k / 32] - 127)
//
// v is e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two a byte, the even k in the low half; s is e8m0, one for
// each 32 along K, 255 a NaN: the OCP microscaling format that model_configs/gpt-oss-120b.json names (mxfp4).
//
// A weight v 2^(s - 127) has two significant bits and fp32's exponents, so it is exact in bf16: the conversion
// instruction takes the scale along, and the bf16 matrix instructions, whose sums keep fp32's bits and whose operands
// may be subnormal, do the rest.  fp16 rows are taken as two bf16 parts, 8 bits and the 3 behind them, which is exact too.
#pragma once

#include "fp8_gemm.h"

namespace moegemm {

constexpr int kMxGroup = 32;
constexpr int kMxBlock = 256;  // K values of a weight row in 128 bytes

struct MxParams {
  const uint16_t* a;    // [rows, k], lda elements between rows
  const uint8_t* w;     // [groups, n, k / 2]
  const uint8_t* sw;    // [groups, n, k / 32]
  void* out;            // [rows, n], or [rows, n / 2] where gated
  const int32_t* offs;
  int64_t lda, swg, ldw, ssg, ssn, ldo;  // weight strides in bytes, rows' and outputs' in elements
  int32_t groups, rows, n, k;
  int32_t n_tiles, out_dtype;
  int32_t first = 0;  // a launch's groups are [first, first + groups)
};

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// Eight weights of a dword, scaled.
__device__ __forceinline__ bf16x8_t mx_weights(uint32_t q, float scale) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3);
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// 2^(s - 127) as the conversion reads it: an exponent field (0 is 2^-127 there, 255 a NaN).
__device__ __forceinline__ float mx_scale(uint32_t s) { return __builtin_bit_cast(float, s << 23); }

// Eight values of a row as bf16 parts that add up to them.
template <class A>
struct RowParts;
template <>
struct RowParts<EBf16> {
  static constexpr int N = 1;
  bf16x8_t v[1];
  __device__ __forceinline__ void set(u32x4_t x) { v[0] = __builtin_bit_cast(bf16x8_t, x); }
};
template <>
struct RowParts<EF16> {
  static constexpr int N = 2;
  bf16x8_t v[2];
  __device__ __forceinline__ void set(u32x4_t x) {
    typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
    typedef uint16_t u16x8_t __attribute__((ext_vector_type(8)));
    const f16x8_t h = __builtin_bit_cast(f16x8_t, x);
    u16x8_t hi, lo;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = (float)h[i];
      const uint32_t top = __builtin_bit_cast(uint32_t, f) & 0xffff0000u;
      hi[i] = (uint16_t)(top >> 16);
      const float rest = f - __builtin_bit_cast(float, top);  // 0 for an infinity, which hi holds whole
      lo[i] = (top & 0x7fffffffu) == 0x7f800000u ? 0 : (uint16_t)(__builtin_bit_cast(uint32_t, rest) >> 16);
    }
    v[0] = __builtin_bit_cast(bf16x8_t, hi);
    v[1] = __builtin_bit_cast(bf16x8_t, lo);
  }
};

// 8 ROWS8 rows of a group by 8 FN weight rows a wave (GATED: 4 FN gate rows and the 4 FN up rows that go with them), WN
// waves along the columns, WK waves that take the K blocks wk, wk + WK, ...
template <class A_, int ROWS8_, int FN_, int WN_, int WK_, bool GATED_>
struct MxStream {
  using A = A_;
  static constexpr int ROWS8 = ROWS8_, FN = FN_, WN = WN_, WK = WK_;
  static constexpr bool GATED = GATED_;
  static constexpr int NT = WN * WK * 64;
  static constexpr int BM = 8 * ROWS8, BN = 8 * FN * WN;
  static constexpr int OUT_COLS = GATED ? BN / 2 : BN;
};

// silu(g) * u in fp32, once rounded by the store.
__device__ __forceinline__ float mx_gated(float g, float u) { return g / (1.0f + __expf(-g)) * u; }

// A wave reads whole 128-byte lines of eight weight rows at a time, straight into registers: lane (q = lane / 16, c = lane %
// 16) holds the 16 bytes, one scale's 32 values, at chunk q + 4 (c / 8) of row c % 8.  As the operand of a 16 x 16 matrix
// instruction, the lanes c >= 8 are eight more "rows": the same ones with the other half of K.  The activations are
// laid out alike, so of the 16 x 16 outputs the two 8 x 8 squares on the diagonal are the halves' sums of eight rows by
// eight rows, and the rest is not used.  That costs half the matrix rate and needs no exchange between lanes.
template <class T>
__global__ void __launch_bounds__(T::NT) mx_stream_kernel(MxParams p) {
  using A = typename T::A;
  constexpr int FN = T::FN, R = T::ROWS8, WK = T::WK, PARTS = RowParts<A>::N;
  __shared__ TileTable table;
  __shared__ float s_sum[WK][T::BM][T::BN + 4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wn = wave % T::WN, wk = wave / T::WN;
  const int c = lane & 15, chunk = (lane >> 4) + 4 * (c >> 3), row8 = c & 7;
  const int f = p.n >> 1;
  build_tile_table(table, p.offs, p.first, p.groups, p.rows, T::BM, p.n_tiles);
  const int units = table.tiles[p.groups - 1];
  const int blocks = (p.k + kMxBlock - 1) / kMxBlock;

  for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
    int lo = 0, hi = p.groups - 1;  // the first group with tiles[i] > unit
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (table.tiles[mid] > unit) hi = mid;
      else lo = mid + 1;
    }
    const int row0 = lo ? table.ends[lo - 1] : table.start, m = table.ends[lo] - row0;
    const int local = unit - (lo ? table.tiles[lo - 1] : 0), m_tiles = (m + T::BM - 1) / T::BM;
    const int tn = local / m_tiles, m0 = (local - tn * m_tiles) * T::BM, n0 = tn * T::OUT_COLS;
    const int e = p.first + lo;

    // Rows past the last are the last again: what they give is not stored.
    const uint8_t* w[FN];
    const uint8_t* s[FN];
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      int n;
      if constexpr (T::GATED)
        n = (i < FN / 2 ? 0 : f) + min(n0 + (wn * (FN / 2) + i % (FN / 2)) * 8 + row8, f - 1);
      else
        n = min(n0 + (wn * FN + i) * 8 + row8, p.n - 1);
      w[i] = p.w + (int64_t)e * p.swg + n * p.ldw + chunk * 16;
      s[i] = p.sw + (int64_t)e * p.ssg + n * p.ssn + chunk;
    }
    const uint16_t* a[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
      a[r] = p.a + ((int64_t)row0 + min(m0 + r * 8 + row8, m - 1)) * p.lda + chunk * kMxGroup;

    f32x4_t acc[R][FN];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < FN; ++i) acc[r][i] = f32x4_t{};
    for (int b = wk; b < blocks; b += WK) {
      const int k0 = b * kMxBlock;
      const bool in = k0 + chunk * kMxGroup < p.k;  // whole groups: K is a multiple of 32
      u32x4_t wv[FN], av[R][4];
      uint32_t sv[FN];
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        wv[i] = u32x4_t{};
        sv[i] = 0;
        if (in) {
          wv[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(w[i] + (k0 >> 1)));
          sv[i] = s[i][k0 >> 5];
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          av[r][x] = u32x4_t{};
          if (in) av[r][x] = *reinterpret_cast<const u32x4_t*>(a[r] + k0 + 8 * x);
        }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        RowParts<A> rows[R];
#pragma unroll
        for (int r = 0; r < R; ++r) rows[r].set(av[r][x]);
#pragma unroll
        for (int i = 0; i < FN; ++i) {
          const bf16x8_t weights = mx_weights(wv[i][x], mx_scale(sv[i]));
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int h = 0; h < PARTS; ++h)
              acc[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(weights, rows[r].v[h], acc[r][i], 0, 0, 0);
        }
      }
    }
    // Lane (q, c) holds weight rows 4 q + j of row c; both halves of K meet, and the WK waves' sums in wave order.
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float v = acc[r][i][j] + __shfl_xor(acc[r][i][j], 40);
          if (lane < 32 && c < 8) s_sum[wk][r * 8 + c][(wn * FN + i) * 8 + (lane >> 4) * 4 + j] = v;
        }
    __syncthreads();
    for (int x = threadIdx.x; x < T::BM * T::OUT_COLS; x += T::NT) {
      const int r = x / T::OUT_COLS, n = x % T::OUT_COLS;
      auto sum = [&](int col) {
        float v = s_sum[0][r][col];
#pragma unroll
        for (int k = 1; k < WK; ++k) v += s_sum[k][r][col];
        return v;
      };
      if (m0 + r >= m || n0 + n >= (T::GATED ? f : p.n)) continue;
      float v;
      if constexpr (T::GATED) {
        const int gate = n / (4 * FN) * 8 * FN + n % (4 * FN);
        v = mx_gated(sum(gate), sum(gate + 4 * FN));
      } else {
        v = sum(n);
      }
      const int64_t to = ((int64_t)row0 + m0 + r) * p.ldo + n0 + n;
      char* out = static_cast<char*>(p.out);
      if (p.out_dtype == DT_F32) store1<EF32>(out + to * 4, v);
      else if (p.out_dtype == DT_BF16) store1<EBf16>(out + to * 2, v);
      else store1<EF16>(out + to * 2, v);
    }
    __syncthreads();
  }
}

// The format's conversions.  A lane takes 8 consecutive values, four lanes a group of 32.
struct MxConvertParams {
  const void* x;   // quantise: values in; dequantise: e2m1 bytes
  uint8_t* q;      // quantise: e2m1 bytes out
  uint8_t* scale;
  void* out;       // dequantise: values out
  int64_t sxr, sqr, ssr;  // row strides: values' in elements, the others' in bytes
  int64_t rows;
  int32_t k;
};

// scale = floor(log2 max|x|) - 2 as an e8m0 byte, at least 0: e2m1's largest power of two is 4.  q = e2m1(x / scale), to
// nearest even, at most 6.  A group that holds a NaN or an infinity gets the scale 255, a NaN.
template <class E, bool VEC>
__global__ void __launch_bounds__(256) mx_quantize_kernel(MxConvertParams p) {
  const int per_row = p.k / 8;
  const int64_t items = p.rows * per_row, step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += step) {  // four lanes of a group go together
    const int64_t row = i / per_row;
    const int col = (int)(i - row * per_row) * 8;
    typename E::raw raw[8];
    const typename E::raw* x = static_cast<const typename E::raw*>(p.x) + row * p.sxr + col;
    if constexpr (VEC) {
      constexpr int N = sizeof(raw) / 16;
      u32x4_t c[N];
#pragma unroll
      for (int j = 0; j < N; ++j) c[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(x) + j);
      __builtin_memcpy(raw, c, sizeof(raw));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) raw[j] = x[j];
    }
    float v[8];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (E::dtype == DT_F32) v[j] = __builtin_bit_cast(float, raw[j]);
      else if constexpr (E::dtype == DT_BF16) v[j] = __builtin_bit_cast(float, (uint32_t)raw[j] << 16);
      else v[j] = (float)__builtin_bit_cast(_Float16, raw[j]);
      top = max(top, abs_bits(v[j]));
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    const int exponent = (int)(top >> 23);  // 255: infinity or NaN; a subnormal maximum's scale is below the least one
    const uint32_t s = exponent == 255 ? 255u : (uint32_t)max(exponent - 2, 0);
    const float scale = mx_scale(exponent == 255 ? 127u : s);
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], scale, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], scale, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], scale, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], scale, 3);
    *reinterpret_cast<uint32_t*>(p.q + row * p.sqr + col / 2) = q;
    if ((col & 31) == 0) p.scale[row * p.ssr + col / 32] = (uint8_t)s;
  }
}

template <class E>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(MxConvertParams p) {
  const int per_row = p.k / 8;
  const int64_t items = p.rows * per_row, step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += step) {
    const int64_t row = i / per_row;
    const int col = (int)(i - row * per_row) * 8;
    const uint32_t q = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(p.x) + row * p.sqr + col / 2);
    const bf16x8_t v = mx_weights(q, mx_scale(p.scale[row * p.ssr + col / 32]));  // exact
    char* out = static_cast<char*>(p.out) + (row * p.k + col) * sizeof(typename E::raw);
    if constexpr (E::dtype == DT_BF16) {
      *MOEGEMM_GLOBAL(u32x4_t, out) = __builtin_bit_cast(u32x4_t, v);
    } else {
      store4<E>(out, f32x4_t{(float)v[0], (float)v[1], (float)v[2], (float)v[3]});
      store4<E>(out + 4 * sizeof(typename E::raw), f32x4_t{(float)v[4], (float)v[5], (float)v[6], (float)v[7]});
    }
  }
}

}  // namespace moegemm
