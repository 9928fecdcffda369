// Products of 16-bit rows with 4-bit weights (MXFP4), and the format's conversions (gfx950).
//
//   C[m, n] = sum_k a[m, k] v[n, k] 2^(s[n, k / 32] - 127)
//
// v is e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two a byte, the even k in the low half; s is e8m0, one
// for each 32 along K, 255 a NaN: the OCP microscaling format that model_configs/gpt-oss-120b.json names (mxfp4).
//
// A weight v 2^(s - 127) has two significant bits and fp32's exponents, so it is exact in bf16: the conversion
// instruction takes the scale along, and the bf16 matrix instructions, whose sums keep fp32's bits and whose operands
// may be subnormal, do the rest.  fp16 rows are taken as two bf16 parts, 8 bits and the 3 behind them, which is exact
// too; fp32 rows as three, their 24 bits, which is exact from 2^-110 up (below, the last part is rounded to 2^-133, bf16's
// least number).  Two would hold 16 bits, which the rounding of some 16-bit outputs shows.  The third costs half as many
// matrix instructions again: 256 rows over 32 experts of [7168, 2048] 62 and 65 us, 16384 over [4096, 7168] 2.55 and 3.4 ms.
#pragma once

#include <type_traits>

#include "fp8_gemm.h"

namespace moegemm {

constexpr int kMxGroup = 32;
constexpr int kMxBlock = 256;  // K values of a weight row in 128 bytes

struct MxParams {
  const void* a;        // [rows, k], lda elements between rows
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

// Eight values of a row as they lie in memory, and as bf16 parts that add up to them.
template <class A>
struct RowPiece {
  static constexpr int LOADS = A::is_f32 ? 2 : 1;
  u32x4_t v[LOADS];
};
template <class A>
struct RowParts {
  static constexpr int N = A::dtype == DT_BF16 ? 1 : A::is_f32 ? 3 : 2;
  bf16x8_t v[N];
  __device__ __forceinline__ void set(const RowPiece<A>& x) {
    if constexpr (A::dtype == DT_BF16) {
      v[0] = __builtin_bit_cast(bf16x8_t, x.v[0]);
    } else {
      typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
      typedef uint16_t u16x8_t __attribute__((ext_vector_type(8)));
      constexpr float kLargest = 0x1.fffffep127f;
      u16x8_t hi, mid, lo;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float f;
        if constexpr (A::is_f32) {
          const uint32_t word = x.v[i >> 2][i & 3];  // a bit cast of the vector's element itself takes the first one
          f = __builtin_canonicalizef(__builtin_bit_cast(float, word));  // quiet, so that hi is a NaN too
        } else {
          f = (float)__builtin_bit_cast(f16x8_t, x.v[0])[i];
        }
        hi[i] = (uint16_t)(__builtin_bit_cast(uint32_t, f) >> 16);
        // Of an infinity or a NaN, which hi holds whole, the median makes the largest number, and the parts behind hi are
        // what is left of that: of an infinity's sign, so that no product of theirs opposes an infinite one.
        const float number = __builtin_amdgcn_fmed3f(f, -kLargest, kLargest);
        const float rest = number - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, number) & 0xffff0000u);
        const uint32_t next = __builtin_bit_cast(uint32_t, rest) & 0xffff0000u;
        mid[i] = (uint16_t)(next >> 16);  // of fp16 all that is left
        if constexpr (A::is_f32) lo[i] = __builtin_bit_cast(uint16_t, (__bf16)(rest - __builtin_bit_cast(float, next)));
      }
      v[0] = __builtin_bit_cast(bf16x8_t, hi);
      v[1] = __builtin_bit_cast(bf16x8_t, mid);
      if constexpr (A::is_f32) v[2] = __builtin_bit_cast(bf16x8_t, lo);
    }
  }
};

// The units of a launch's groups, in LDS behind the kernel's other arrays: cumulative counts of ceil(m / bm) * n_tiles,
// and the groups' rows.
constexpr int kMxTable = 1024;
struct MxTable {
  int32_t* units;
  int32_t* ends;  // offsets, clamped
  int32_t* sums;  // [16]
  int32_t* start;  // the first group's first row
  __device__ __forceinline__ MxTable(int32_t* at, int groups) : units(at + 17), ends(at + 17 + groups), sums(at), start(at + 16) {}
  static size_t bytes(int groups) { return (17 + 2 * (size_t)groups) * sizeof(int32_t); }
};

// Sums stop at INT32_MAX, which only overlapping groups of decreasing offsets reach.
__device__ __forceinline__ uint32_t add_units(uint32_t a, uint32_t b) { return min(a + b, (uint32_t)INT32_MAX); }

// Every thread of the workgroup calls it; returns the number of units and ends with a barrier.
template <int NT>
__device__ __forceinline__ int mx_table(const MxTable& table, const MxParams& p, int bm) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t base = 0;
  for (int g0 = 0; g0 < p.groups; g0 += NT) {
    const int g = g0 + (int)threadIdx.x;
    int m = 0, row0 = 0;
    if (g < p.groups) row0 = group_rows(p.offs, p.rows, p.first + g, m);
    if (g < p.groups) table.ends[g] = p.offs ? min(max(p.offs[p.first + g], 0), p.rows) : p.rows;  // the next group's first row
    if (g == 0) *table.start = row0;
    uint32_t count = (uint32_t)min((int64_t)((m + bm - 1) / bm) * p.n_tiles, (int64_t)INT32_MAX);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t below = (uint32_t)__shfl_up((int)count, d);
      count = lane >= d ? add_units(count, below) : count;
    }
    if (lane == 63) table.sums[wave] = (int32_t)count;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
      const uint32_t n = (uint32_t)table.sums[w];
      if (w < wave) count = add_units(count, n);
    }
    if (g < p.groups) table.units[g] = (int32_t)add_units(base, count);
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) base = add_units(base, (uint32_t)table.sums[w]);
    __syncthreads();
  }
  return (int)base;
}

// The group of a unit, its rows and the unit's place among the group's.
__device__ __forceinline__ int mx_find(const MxTable& table, int groups, int unit, int& row0, int& m, int& local) {
  int lo = 0, hi = groups - 1;  // the first group with units[i] > unit
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (table.units[mid] > unit) hi = mid;
    else lo = mid + 1;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  row0 = __builtin_amdgcn_readfirstlane(lo ? table.ends[lo - 1] : *table.start);
  m = __builtin_amdgcn_readfirstlane(table.ends[lo]) - row0;
  local = unit - __builtin_amdgcn_readfirstlane(lo ? table.units[lo - 1] : 0);
  return lo;
}

// ROWS rows of a group by 8 FN weight rows a wave (GATED: 4 FN gate rows and the 4 FN up rows that go with them), and
// WN waves along the columns, which share the rows through LDS, or WK waves that take a part of K each.
template <class A_, int ROWS_, int FN_, int WN_, int WK_, bool GATED_>
struct MxStream {
  using A = A_;
  static constexpr int FN = FN_, WN = WN_, WK = WK_;
  static constexpr bool GATED = GATED_, SHARED = WN > 1;
  static constexpr int NT = WN * WK * 64;
  static constexpr int BM = ROWS_, BN = 8 * FN * WN;
  static constexpr bool EIGHT = BM == 8;
  static constexpr int FM = EIGHT ? 1 : BM / 16, TILES = EIGHT ? FN : FN / 2;  // of 16 x 16 sums
  static constexpr int HALVES = EIGHT ? 1 : 2;                                 // pieces of a row a lane needs of a block, by four
  static constexpr int OUT_COLS = GATED ? BN / 2 : BN;
  static constexpr int PARTS = RowParts<A>::N;
  static constexpr int CHUNK_BLOCKS = PARTS == 1 && BM <= 32 ? 2 : 1;  // K blocks of the rows in LDS
  static constexpr int CHUNK = CHUNK_BLOCKS * kMxBlock;
  static constexpr int ROW_BYTES = CHUNK * 2 + 16;       // 16 bytes more: rows' pieces on all banks
  static constexpr int STAGE_BYTES = BM * ROW_BYTES;     // of one part
  static constexpr int ES = sizeof(typename A::raw);
  static constexpr int COPIES = BM * CHUNK / 8 / NT;     // pieces of a stage a thread
  // One where two would leave LDS for one workgroup a CU (16384 fp32 rows over 32 experts of [4096, 7168] 3.8 and 3.4 ms).
  static constexpr int STAGES = PARTS == 3 && BM == 32 ? 1 : 2;
  static constexpr int ROWS_BYTES = SHARED ? STAGES * PARTS * STAGE_BYTES : 0;
  static constexpr int SUM_BYTES = WK * BM * (BN + 4) * 4;
  static constexpr int LDS_BYTES = ROWS_BYTES > SUM_BYTES ? ROWS_BYTES : SUM_BYTES;  // the sums where the rows were
  // Workgroups a CU, and waves a SIMD that the registers allow.  Where rows are shared two: a third leaves too few
  // registers for the blocks ahead, and the units come out uneven (256 rows over 32 experts, 8 a unit, 127 us and 135);
  // rows of two or three parts, which have no more than one block ahead, three up to 16 a unit (fp16 116 and 101 us, over
  // [7168, 2048] 59 and 50).  Units of one wave's width two as well, 16 rows of three parts one, whose registers spill else
  // (32 rows of [4096, 7168] 25.8 and 22.6 us), and up to four's worth of workgroups that wait (Gate+Up of four rows over
  // 128 experts of [5760, 2880] by two 11.6 us, by four 10.5, by eight 10.7).
  static constexpr int MIN_WAVES = SHARED && PARTS > 1 && BM <= 16 ? 3 : !SHARED && PARTS == 3 && !EIGHT ? 1 : 2;
  static constexpr int PER_CU = SHARED ? MIN_WAVES : 4;
  // Blocks of weights on their way.  256 rows over 32 experts of [4096, 7168] 86 us with three, 89 with one; over
  // [7168, 2048] 56 and 60.  Rows of two parts, whose matrix instructions take twice as long, fp32 by two of their parts: 128 and 127, 71 and
  // 65; 2048 rows, 64 a unit, over [4096, 7168] 219 and 210; waves with a part of K, one row of [5760, 2880] 6.6 and
  // 5.7.
  static constexpr int AHEAD = SHARED && PARTS == 1 && BM <= 32 ? 3 : 1;
  static_assert(4 % (AHEAD + 1) == 0, "a block's registers are known");
  static_assert(EIGHT || BM % 16 == 0, "whole matrix instructions");
  static_assert(FN % 2 == 0, "weight rows go in pairs of eights");
  static_assert(WN == 1 || WK == 1, "columns or K");
  static_assert(!SHARED || BM * CHUNK / 8 % NT == 0, "whole copies");
  static_assert(LDS_BYTES + 17 * 4 + 8 * kMxTable <= 160 * 1024, "LDS of one CU");
};

// silu(g) * u in fp32, once rounded by the store.
__device__ __forceinline__ float mx_gated(float g, float u) { return g / (1.0f + __expf(-g)) * u; }

typedef __amdgpu_buffer_rsrc_t mx_rsrc_t;
__device__ __forceinline__ mx_rsrc_t mx_resource(const void* base, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}
template <bool ONCE = false>  // non-temporal
__device__ __forceinline__ u32x4_t mx_load16(mx_rsrc_t r, uint32_t offset) {
  return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, (int)offset, 0, ONCE ? 2 : 0));
}

// A wave reads whole 128-byte lines of eight weight rows at a time, straight into registers: lane (q = lane / 16, c =
// lane % 16) holds the 16 bytes, one scale's 32 values, at chunk q + 4 (c / 8) of row c % 8.  The 16 x 16 matrix
// instructions want one row a lane c, and one K for all rows: lanes c + 8 of eight rows change places with lanes c of
// the next eight (a DPP move of each dword), which gives sixteen rows' first halves of the block, and their second
// halves.  For up to EIGHT rows the weights stay where they are: lanes c >= 8 are the same eight weight rows with the
// other half of K, the activations are laid out alike, and of the 16 x 16 sums the two 8 x 8 squares on the diagonal
// are the halves' sums; as many matrix instructions, half the rows to load and split.
//
// The next blocks' weights are on their way while one is multiplied, and the scales of the next sixteen: a lane loads
// 16 of a row's 128 bytes and the lanes of the row exchange them, since byte loads of each lane's own cost as many
// requests as the weights (256 rows over 32 experts of [4096, 7168]: bytes 115 us, four at a time 95, 16 92).  Offsets
// past a resource's bytes, which rows past the last and K blocks past the end are given, read zeros and fetch nothing.
//
// ONCE: weights pass the caches by.  That is faster where a line belongs to one block of one row that one unit reads
// (256 rows over 32 experts of [4096, 7168]: 86 us, kept 102), and slower where rows begin inside a line, whose other
// part the next block or row reads soon after (256 rows over 128 experts of [5760, 2880]: 255 us, kept 232), or where a
// group's other units read the weights too (2048 rows over 32 of [7168, 2048], 32 a unit: 152 us, kept 134).
//
// Decode is bound by HBM's reads: 256 bf16 rows over 32 experts of [4096, 7168], 0.50 GB, 88 to 92 us, 5.4 to 5.7 TB/s;
// 4 rows of 128 experts of [5760, 2880], 35 MB, 11.8 us, of which the launch, one memory latency after the other and
// the table are an estimated half.  fp32 rows cost their split and three times the matrix instructions: vector and
// matrix instructions fill nearly nine tenths of the cycles, 256 by [7168, 2048] 61 to 67 us, bf16 53 (0.25 GB, 4.8
// TB/s).  From 64 rows a group on the matrix pipes and the conversions are the bound: 16384 rows over 32 experts of
// [4096, 7168] 1191 us, 0.81 PFLOP/s.
template <class T, bool ONCE>
__global__ void __launch_bounds__(T::NT, T::MIN_WAVES) mx_stream_kernel(MxParams p) {
  using A = typename T::A;
  constexpr int FM = T::FM, FN = T::FN, WK = T::WK, PARTS = T::PARTS, TILES = T::TILES, HALVES = T::HALVES;
  __shared__ __attribute__((aligned(16))) char smem[T::LDS_BYTES];
  extern __shared__ int32_t s_table[];
  const MxTable table(s_table, p.groups);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wn = wave % T::WN, wk = wave / T::WN;
  const int c = lane & 15, quad = lane >> 4, chunk = quad + 4 * (c >> 3), row8 = c & 7;
  const int f = p.n >> 1;
  const int blocks = (p.k + kMxBlock - 1) / kMxBlock, part = (blocks + WK - 1) / WK;
  const int first_b = min(wk * part, blocks), end_b = min(first_b + part, blocks);  // the wave's K blocks
  const int scales = p.k / kMxGroup;                                                // of a row
  const uint32_t units = (uint32_t)mx_table<T::NT>(table, p, T::BM);

  constexpr int WAVE_ROWS = T::GATED ? 4 * FN : 8 * FN;  // weight rows of one resource
  constexpr int AHEAD = T::AHEAD;
  const int byte_shift = (chunk & 3) * 8;
  const int out_cols = T::GATED ? f : p.n;
  // The unit whose loads are issued.
  int first_n = 0, valid_m = 0, n0 = 0;
  int64_t first_row = 0;
  mx_rsrc_t rw, rw2, ra;
  const uint8_t* s = nullptr;
  const uint32_t w_lane = (uint32_t)row8 * (uint32_t)p.ldw + chunk * 16;
  auto set_unit = [&](int unit) {
    int row0, m, local;
    const int e = p.first + mx_find(table, p.groups, unit, row0, m, local);
    const int m_tiles = (m + T::BM - 1) / T::BM, tn = local / m_tiles, m0 = (local - tn * m_tiles) * T::BM;
    first_row = (int64_t)row0 + m0;
    valid_m = min(T::BM, m - m0);
    n0 = tn * T::OUT_COLS;
    first_n = n0 + wn * WAVE_ROWS;
    const int valid_n = min(WAVE_ROWS, out_cols - first_n);
    const uint8_t* w = p.w + (int64_t)e * p.swg + (int64_t)first_n * p.ldw;
    const int64_t w_bytes = valid_n > 0 ? (valid_n - 1) * p.ldw + (p.k >> 1) : 0;
    rw = mx_resource(w, w_bytes);
    rw2 = T::GATED ? mx_resource(w + f * p.ldw, w_bytes) : rw;
    ra = mx_resource(static_cast<const char*>(p.a) + first_row * p.lda * T::ES, ((valid_m - 1) * p.lda + p.k) * T::ES);
    s = p.sw + (int64_t)e * p.ssg;
  };
  auto load = [&](u32x4_t (&q)[FN], int b) {
    const bool in = b < end_b && b * kMxBlock + chunk * kMxGroup < p.k;  // whole groups: K is a multiple of 32
    const uint32_t wo = in ? w_lane + (uint32_t)b * (kMxBlock / 2) : kOutOfRange;
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      const bool up = T::GATED && i >= FN / 2;
      q[i] = mx_load16<ONCE>(up ? rw2 : rw, wo + (uint32_t)((up ? i - FN / 2 : i) * 8) * (uint32_t)p.ldw);
    }
  };
  // The lane's 16 of the 128 bytes of blocks b to b + 15; zeros past the row's end, where nothing is read.
  auto load_scales = [&](u32x4_t (&v)[FN], int b) {
    const int want = b * (kMxBlock / kMxGroup) + chunk * 16, at = max(min(want, scales - 16), 0);
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      const bool up = T::GATED && i >= FN / 2;
      const int n = min(first_n + (up ? i - FN / 2 : i) * 8 + row8, out_cols - 1) + (up ? f : 0);
      const uint8_t* from = s + n * p.ssn + at;
      if (scales >= 16) {
        __builtin_memcpy(&v[i], from, 16);
      } else {
        v[i] = u32x4_t{};
        for (int j = 0; j < scales; ++j) {
          const uint32_t byte = (uint32_t)from[j] << (8 * (j & 3));
#pragma unroll
          for (int x = 0; x < 4; ++x) v[i][x] |= j >> 2 == x ? byte : 0;
        }
      }
    }
  };
  // The same once they are here: moved to where the lane's bytes would be if the row went on.
  auto settle_scales = [&](u32x4_t (&v)[FN], int b) {
    const int want = b * (kMxBlock / kMxGroup) + chunk * 16, past = want - max(min(want, scales - 16), 0);
    if (__ballot(past > 0) == 0) return;
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      u32x4_t x = v[i];
      if (past & 8) x = u32x4_t{x[2], x[3], 0, 0};
      if (past & 4) x = u32x4_t{x[1], x[2], x[3], 0};
      const uint32_t bytes = past & 3;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = past >= 16 ? 0 : __builtin_amdgcn_alignbyte(j < 3 ? x[j + 1] : 0, x[j], bytes);
    }
  };
  f32x4_t acc[FM][TILES];
  // Block `at` of the sixteen whose scales are at hand: byte 8 at + chunk of the row's 128, which lane at / 2 of the
  // row's holds.
  auto multiply = [&](const u32x4_t (&q)[FN], const u32x4_t (&bytes)[FN], int at, int odd, auto&& rows_of) {
    const int other = at >> 1, from = ((other & 3) * 16 + (other >> 2) * 8 + row8) * 4;
    uint32_t scale[FN];
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      const uint32_t low = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)bytes[i][2 * odd]);
      const uint32_t high = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)bytes[i][2 * odd + 1]);
      scale[i] = (chunk < 4 ? low : high) >> byte_shift & 0xff;
    }
    // Of two eights of rows: all sixteen's first halves of the block, and their second.
    auto first = [](uint32_t a, uint32_t b) {
      return (uint32_t)__builtin_amdgcn_update_dpp((int)a, (int)b, 0x128, 0xf, 0xc, false);  // row_ror:8 into lanes 8 to 15
    };
    auto second = [](uint32_t a, uint32_t b) {
      return (uint32_t)__builtin_amdgcn_update_dpp((int)b, (int)a, 0x128, 0xf, 0x3, false);  // into lanes 0 to 7
    };
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      RowParts<A> rows[FM][HALVES];
#pragma unroll
      for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int half = 0; half < HALVES; ++half) rows_of(rows[m][half], m, half, x);
      if constexpr (T::EIGHT) {
#pragma unroll
        for (int i = 0; i < FN; ++i) {
          const bf16x8_t weights = mx_weights(q[i][x], mx_scale(scale[i]));
#pragma unroll
          for (int h = 0; h < PARTS; ++h)
            acc[0][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(weights, rows[0][0].v[h], acc[0][i], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int i = 0; i < FN; i += 2) {
          const uint32_t a = q[i][x], b = q[i + 1][x];
          const bf16x8_t weights[2] = {mx_weights(first(a, b), mx_scale(first(scale[i], scale[i + 1]))),
                                       mx_weights(second(a, b), mx_scale(second(scale[i], scale[i + 1])))};
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int m = 0; m < FM; ++m)
#pragma unroll
              for (int h = 0; h < PARTS; ++h)
                acc[m][i / 2] =
                    __builtin_amdgcn_mfma_f32_16x16x32_bf16(weights[half], rows[m][half].v[h], acc[m][i / 2], 0, 0, 0);
        }
      }
    }
  };
  // Shared rows go through registers to LDS, CHUNK values at a time and one chunk ahead, split into their parts on the
  // way; a wave that has its own part of K loads them as it needs them.
  constexpr uint32_t ES = T::ES;
  auto load_piece = [&](RowPiece<A>& v, uint32_t offset) {
#pragma unroll
    for (int l = 0; l < RowPiece<A>::LOADS; ++l) v.v[l] = mx_load16(ra, offset + l * 16);
  };
  RowPiece<A> piece[T::SHARED ? T::COPIES : 1], av[T::SHARED ? 1 : 2][FM][HALVES][4];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int j = 0; j < T::COPIES; ++j) {
      const int at = threadIdx.x + j * T::NT, row = at / (T::CHUNK / 8), col = at % (T::CHUNK / 8);
      const uint32_t offset = ((uint32_t)row * (uint32_t)p.lda + (uint32_t)(k0 + col * 8)) * ES;
      load_piece(piece[j], row < valid_m && k0 + col * 8 < p.k ? offset : kOutOfRange);
    }
  };
  auto put = [&](int stage) {
#pragma unroll
    for (int j = 0; j < T::COPIES; ++j) {
      const int at = threadIdx.x + j * T::NT, row = at / (T::CHUNK / 8), col = at % (T::CHUNK / 8);
      RowParts<A> parts;
      parts.set(piece[j]);
#pragma unroll
      for (int h = 0; h < PARTS; ++h)
        *reinterpret_cast<bf16x8_t*>(smem + (stage * PARTS + h) * T::STAGE_BYTES + row * T::ROW_BYTES + col * 16) = parts.v[h];
    }
  };
  const int a_row = T::EIGHT ? row8 : c, a_chunk = T::EIGHT ? chunk : quad;  // of the lane, among 8 or 16
  const uint32_t a_lane = ((uint32_t)a_row * (uint32_t)p.lda + a_chunk * kMxGroup) * ES;
  auto fetch_own = [&](RowPiece<A> (&v)[FM][HALVES][4], int b) {
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
      for (int half = 0; half < HALVES; ++half) {
        const int k0 = b * kMxBlock + half * (kMxBlock / 2);
        const bool in = b < end_b && k0 + a_chunk * kMxGroup < p.k && m * 16 + a_row < valid_m;
        const uint32_t ao = a_lane + ((uint32_t)(m * 16) * (uint32_t)p.lda + (uint32_t)k0) * ES;
#pragma unroll
        for (int x = 0; x < 4; ++x) load_piece(v[m][half][x], in ? ao + x * 8 * ES : kOutOfRange);
      }
  };
  // Waves meet without waiting for what is on its way from memory.
  auto meet = [] {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    compiler_fence();
  };
  const uint32_t frag = (uint32_t)a_row * T::ROW_BYTES + a_chunk * (kMxGroup * 2);

  u32x4_t q[AHEAD + 1][FN];
  u32x4_t bytes[FN], next_bytes[FN];  // scales of sixteen blocks
  auto start = [&](int unit) {
    set_unit(unit);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) load(q[j], first_b + j);
    load_scales(bytes, first_b);
    if constexpr (T::SHARED) fetch(0);
    else fetch_own(av[0], first_b);
  };
  uint32_t unit = blockIdx.x;  // one past INT32_MAX units is past a signed one's range
  if (unit >= units) return;
  start(unit);
  while (true) {
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
      for (int i = 0; i < TILES; ++i) acc[m][i] = f32x4_t{};
    if constexpr (T::SHARED) {
      put(0);
      meet();
    }
    settle_scales(bytes, first_b);
    constexpr int CB = T::CHUNK_BLOCKS;
    for (int b0 = first_b; b0 < end_b; b0 += 4) {
      const int rel = b0 - first_b & 15;
      if (rel == 8) load_scales(next_bytes, b0 + 8);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int b = b0 + j;
        if (b >= end_b) break;
        if constexpr (T::SHARED) {
          const int stage = T::STAGES == 1 ? 0 : j / CB & 1, place = j % CB;
          if (place == 0) fetch((b + CB) * kMxBlock);
          load(q[(j + AHEAD) % (AHEAD + 1)], b + AHEAD);
          multiply(q[j % (AHEAD + 1)], bytes, rel + j, j & 1, [&](RowParts<A>& rows, int m, int half, int x) {
#pragma unroll
            for (int h = 0; h < PARTS; ++h)
              rows.v[h] = *reinterpret_cast<const bf16x8_t*>(smem + (stage * PARTS + h) * T::STAGE_BYTES + frag +
                                                            m * 16 * T::ROW_BYTES + place * (kMxBlock * 2) +
                                                            half * kMxBlock + x * 16);
          });
          if (place == CB - 1 && b + 1 < end_b) {
            if constexpr (T::STAGES == 1) meet();
            put(T::STAGES == 1 ? 0 : stage ^ 1);
            meet();
          }
        } else {
          load(q[(j + AHEAD) % (AHEAD + 1)], b + AHEAD);
          fetch_own(av[(j + 1) & 1], b + 1);
          multiply(q[j % (AHEAD + 1)], bytes, rel + j, j & 1, [&](RowParts<A>& rows, int m, int half, int x) {
            rows.set(av[j & 1][m][half][x]);
          });
        }
      }
      if (rel == 12) {
#pragma unroll
        for (int i = 0; i < FN; ++i) bytes[i] = next_bytes[i];
        settle_scales(bytes, b0 + 4);
      }
    }

    // The next unit's loads go out before this one's results.
    const int done_m = valid_m, done_n = n0;
    const int64_t done_row = first_row;
    unit += gridDim.x;
    if (unit < units) start(unit);

    // Lane (q, c) holds weight rows 4 q + j of sixteen, of row c, or of EIGHT both halves of K meet; the WK waves' sums
    // are added in wave order.
    if constexpr (T::SHARED) meet();  // the sums go where the rows are
    float* sums = reinterpret_cast<float*>(smem);
    constexpr int LD = T::BN + 4;
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        f32x4_t v = acc[m][i];
        if constexpr (T::EIGHT) {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] += __shfl_xor(v[j], 40);
        }
        if (!T::EIGHT || (quad < 2 && c < 8))
          *reinterpret_cast<f32x4_t*>(sums + (wk * T::BM + m * 16 + c) * LD + wn * 8 * FN + i * (8 * HALVES) + quad * 4) = v;
      }
    meet();
    for (int x = threadIdx.x; x < T::BM * T::OUT_COLS; x += T::NT) {
      const int r = x / T::OUT_COLS, n = x % T::OUT_COLS;
      auto sum = [&](int col) {
        float v = sums[r * LD + col];
#pragma unroll
        for (int k = 1; k < WK; ++k) v += sums[(k * T::BM + r) * LD + col];
        return v;
      };
      if (r >= done_m || done_n + n >= out_cols) continue;
      float v;
      if constexpr (T::GATED) {
        const int gate = n / (4 * FN) * 8 * FN + n % (4 * FN);
        v = mx_gated(sum(gate), sum(gate + 4 * FN));
      } else {
        v = sum(n);
      }
      const int64_t to = (done_row + r) * p.ldo + done_n + n;
      char* out = static_cast<char*>(p.out);
      if (p.out_dtype == DT_F32) store1<EF32>(out + to * 4, v);
      else if (p.out_dtype == DT_BF16) store1<EBf16>(out + to * 2, v);
      else store1<EF16>(out + to * 2, v);
    }
    if (unit >= units) break;
    meet();
  }
}

// The format's conversions.  An item is 16 bytes of values, so that a wave's loads and stores of them cover whole
// lines: 8 values of 16 bits or 4 of 32, and 4 or 8 lanes a group of 32.  Each thread has four items on their way.
struct MxConvertParams {
  const void* x;   // quantise: values in; dequantise: e2m1 bytes
  uint8_t* q;      // quantise: e2m1 bytes out
  uint8_t* scale;
  void* out;       // dequantise: values out
  int64_t sxr, sqr, ssr;  // row strides: values' in elements, the others' in bytes
  int64_t rows;
  int64_t k;
};
template <class E>
struct MxItem {
  static constexpr int VALUES = 16 / sizeof(typename E::raw);
  using packed_t = std::conditional_t<VALUES == 8, uint32_t, uint16_t>;
};
constexpr int kMxItems = 4;
// Where item i lies: its row, and its first column.
template <class E>
__device__ __forceinline__ void mx_item(const MxConvertParams& p, int64_t i, int64_t& row, int64_t& col) {
  const int64_t per_row = p.k / MxItem<E>::VALUES;
  row = p.rows == 1 ? 0 : i / per_row;
  col = (i - row * per_row) * MxItem<E>::VALUES;
}

// scale = floor(log2 max|x|) - 2 as an e8m0 byte, at least 0: e2m1's largest power of two is 4.  q = e2m1(x / scale),
// to nearest even, at most 6.  A group that holds a NaN or an infinity gets the scale 255, a NaN. Bound by HBM: 8 x
// [5760, 2880] in fp32 95 to 98 us, 6.1 to 6.3 TB/s read and written.  Values are read once, past the caches.
template <class E, bool VEC>
__global__ void __launch_bounds__(256) mx_quantize_kernel(MxConvertParams p) {
  using raw_t = typename E::raw;
  constexpr int V = MxItem<E>::VALUES;
  const int64_t items = p.rows * (p.k / V), step = (int64_t)gridDim.x * 256 * kMxItems;
  for (int64_t i0 = (int64_t)blockIdx.x * 256 * kMxItems + threadIdx.x; i0 < items; i0 += step) {  // a group's lanes go together
    u32x4_t chunk[kMxItems];
#pragma unroll
    for (int u = 0; u < kMxItems; ++u) {
      int64_t row, col;
      mx_item<E>(p, min(i0 + u * 256, items - 1), row, col);
      const raw_t* x = static_cast<const raw_t*>(p.x) + row * p.sxr + col;
      if constexpr (VEC) {
        chunk[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(x));
      } else {
        raw_t raw[V];
#pragma unroll
        for (int j = 0; j < V; ++j) raw[j] = x[j];
        __builtin_memcpy(&chunk[u], raw, 16);
      }
    }
#pragma unroll
    for (int u = 0; u < kMxItems; ++u) {
      if (i0 + u * 256 >= items) break;
      int64_t row, col;
      mx_item<E>(p, i0 + u * 256, row, col);
      raw_t raw[V];
      __builtin_memcpy(raw, &chunk[u], 16);
      float v[V];
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if constexpr (E::dtype == DT_F32) v[j] = __builtin_bit_cast(float, raw[j]);
        else if constexpr (E::dtype == DT_BF16) v[j] = __builtin_bit_cast(float, (uint32_t)raw[j] << 16);
        else v[j] = (float)__builtin_bit_cast(_Float16, raw[j]);
        top = max(top, abs_bits(v[j]));
      }
#pragma unroll
      for (int d = 1; d < kMxGroup / V; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
      const int exponent = (int)(top >> 23);  // 255: infinity or NaN; a subnormal maximum's scale is below the least one
      const uint32_t s = exponent == 255 ? 255u : (uint32_t)max(exponent - 2, 0);
      const float scale = mx_scale(exponent == 255 ? 127u : s);
      uint32_t q = 0;
      q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], scale, 0);
      q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], scale, 1);
      if constexpr (V == 8) {
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], scale, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], scale, 3);
      }
      *reinterpret_cast<typename MxItem<E>::packed_t*>(p.q + row * p.sqr + col / 2) = (typename MxItem<E>::packed_t)q;
      if ((col & 31) == 0) p.scale[row * p.ssr + col / 32] = (uint8_t)s;
    }
  }
}

// Each value is exact in bf16.  Bound by HBM: 8 x [5760, 2880] to fp32 84 us, 7.2 TB/s read and written.  Stores go
// past the caches at every size: to bf16, 17 MB 4.6 us, kept 5.0; 133 MB 24.6 and 25.1; 265 MB 48 and 59; to fp32, 531
// MB 85 and 106.  A copy of the values right behind it gains less from kept ones (17 MB 16.4 and 15.0, 265 MB 158 and
// 162).
template <class E>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(MxConvertParams p) {
  using raw_t = typename E::raw;
  using packed_t = typename MxItem<E>::packed_t;
  constexpr int V = MxItem<E>::VALUES;
  const int64_t items = p.rows * (p.k / V), step = (int64_t)gridDim.x * 256 * kMxItems;
  for (int64_t i0 = (int64_t)blockIdx.x * 256 * kMxItems + threadIdx.x; i0 < items; i0 += step) {
    uint32_t q[kMxItems], s[kMxItems];
#pragma unroll
    for (int u = 0; u < kMxItems; ++u) {
      int64_t row, col;
      mx_item<E>(p, min(i0 + u * 256, items - 1), row, col);
      q[u] = *reinterpret_cast<const packed_t*>(static_cast<const uint8_t*>(p.x) + row * p.sqr + col / 2);
      s[u] = p.scale[row * p.ssr + col / 32];
    }
#pragma unroll
    for (int u = 0; u < kMxItems; ++u) {
      if (i0 + u * 256 >= items) break;
      const bf16x8_t v = mx_weights(q[u], mx_scale(s[u]));  // exact
      u32x4_t out;
      if constexpr (E::dtype == DT_BF16) {
        out = __builtin_bit_cast(u32x4_t, v);
      } else {
        raw_t raw[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if constexpr (E::is_f32) raw[j] = __builtin_bit_cast(uint32_t, (float)v[j]);
          else raw[j] = __builtin_bit_cast(uint16_t, (_Float16)(float)v[j]);
        }
        __builtin_memcpy(&out, raw, 16);
      }
      __builtin_nontemporal_store(out, reinterpret_cast<u32x4_t*>(p.out) + i0 + u * 256);
    }
  }
}

}  // namespace moegemm
