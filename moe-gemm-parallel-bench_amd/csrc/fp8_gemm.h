// Products of e4m3 operands with one fp32 scale for each block of 128 along K (gfx950).
//
//   C[m, n] = sum_b sa[m, b] sw[n / 128, b] * (sum_{k in block b} a[m, k] w[n, k])
//
// a [rows, K] carries a scale for each row and block of 128 columns, w [N, K] (a linear layer's
// weight) one for each 128 x 128 block.  The inner sum runs on the matrix cores from a zero
// accumulator; one fp32 FMA per output and block adds it, scaled, to the running sum.  Scales are
// arbitrary fp32 numbers, so the matrix instructions' own power-of-two block scales cannot carry them.
//
// Two ways to form the inner sum:
//  * exact: e4m3 values are widened to bf16 (exactly) in registers and multiplied with the bf16
//    instructions, whose sums keep fp32's bits: 2^16 + 2^-7 comes back whole;
//  * FAST: the 8-bit instructions (32x32x64), at twice the rate.  They add eight products at a time
//    and drop what is below 2^-13 of the largest (2^16 + 8 came back whole, 2^16 + 4 as 2^16, where
//    both products are among the same eight), then in fp32.  Fewer than 32 bits, so the caller has to
//    ask for it; an output is off by at most 2^-10 sum |a w|.
//
// Operands are swapped (D^T = W A^T, as in gemm_kernel.h): a lane owns one output row m, so a
// block's scale is one value per lane and fragment, and four consecutive columns n per register
// quad, which the epilogue stores as vectors.  Within a block the order of k does not matter, so
// fragments take their 32 bytes as two 16-byte chunks 64 bytes apart (or as the LDS swizzle likes
// them), the same two for both operands.
//
// Rows are grouped by cumulative end offsets on the device as in MODE_OFFSETS (gemm_kernel.h), or
// form one group (offs null).  Two kernels:
//  * Fp8Tile (prefill): operands reach LDS by DMA, one 128-byte K slice (= one scale block) per
//    stage, 16-byte chunks XOR-swizzled, read with ds_read_b128;
//  * Fp8Stream (decode, few rows a group): each wave streams weights through a ring of its own in LDS, every
//    byte read once where a group has no more rows than a unit (16 or 32), and once for each 16 or 32 rows
//    of it otherwise.  Exact sums only: HBM is the bound, and widening costs no time.
#pragma once

#include "gemm_fast.h"

namespace moegemm {

typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));
typedef int32_t i32x8_t __attribute__((ext_vector_type(8)));

constexpr int kScaleBlock = 128;
constexpr float kE4m3Max = 448.0f;
constexpr float kAmaxFloor = 0x1p-96f;  // amax of a block of zeros: a finite scale and its reciprocal

struct Fp8Params {
  const uint8_t* a;   // [rows, k], lda bytes between rows
  const float* sa;    // [rows, blocks of k]
  const uint8_t* w;   // [groups, n, k]
  const float* sw;    // [groups, blocks of n, blocks of k]
  void* out;          // [rows, n] (plain) or e4m3 [rows, n / 2] (gated)
  float* out_scale;   // gated: [rows, blocks of n / 2]
  const int32_t* offs;
  int64_t lda, sam, sak;            // scale strides in elements
  int64_t swg, ldw, ssg, ssn, ssk;  // weight strides in bytes, its scales' in elements
  int64_t ldo, osm, osk;            // output row pitch in elements, output scale strides
  int32_t groups, rows, n, k;
  int32_t n_tiles;                  // column tiles (the launch's)
  int32_t first = 0;  // tile kernels: a launch's groups are [first, first + groups), its rounds start at `round`
  int32_t round = 0;
};

// Rows of group e: [row0, row0 + m), offsets clamped to [0, rows], a decreasing offset empty.
__device__ __forceinline__ int group_rows(const int32_t* offs, int rows, int e, int& m) {
  if (!offs) {
    m = rows;
    return 0;
  }
  const int lo = e == 0 ? 0 : min(max(offs[e - 1], 0), rows);
  const int hi = min(max(offs[e], 0), rows);
  m = max(hi - lo, 0);
  return lo;
}

struct GroupTile {
  int e, row0, m, tm, tn;
  int part;  // first row in the tile (see build_tile_list)
};

__device__ __forceinline__ float uniform(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}

// The lane, computed where it is used.  The tile loops' lookups, tails and epilogues depend on the lane and not on the
// tile: hoisted out of the loop, their offsets took a hundred spilled registers.
__device__ __forceinline__ int lane_here() {
  uint32_t none = 0;
  asm volatile("" : "+s"(none));
  return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, none));
}

__device__ __forceinline__ int64_t value_of(int64_t x, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(lane * 4, (int)(uint32_t)x);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(lane * 4, (int)(uint32_t)((uint64_t)x >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// The tiles of a launch's groups, ceil(m / bm) * n_tiles each, in LDS: a search over the offsets in memory would load them
// into vector registers and wait for every copy and store in flight, which a loop that prefetches across tiles
// must not.  A call with more groups is several launches.
constexpr int kTableGroups = 768;
struct TileTable {
  int32_t tiles[kTableGroups];  // cumulative tile counts
  int32_t ends[kTableGroups];   // offsets, clamped
  int32_t start;                // the first group's first row
};

// Groups [first, first + groups).  Every thread of the workgroup calls it; ends with a barrier.
__device__ __forceinline__ void build_tile_table(TileTable& table, const int32_t* offs, int first, int groups, int rows,
                                                 int bm, int n_tiles) {
  const int lane = threadIdx.x & 63;
  if (threadIdx.x < 64) {
    int64_t base = 0;
    for (int chunk = 0; chunk < groups; chunk += 64) {
      const int i = chunk + lane;
      int m = 0, row0 = 0;
      if (i < groups) row0 = group_rows(offs, rows, first + i, m);
      int64_t sum = (int64_t)((m + bm - 1) / bm) * n_tiles;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int64_t below = value_of(sum, lane - d);
        if (lane >= d) sum += below;
      }
      sum = min(base + sum, (int64_t)INT32_MAX);  // overlapping groups of decreasing offsets
      if (i < groups) {
        table.tiles[i] = (int32_t)sum;
        table.ends[i] = offs ? min(max(offs[first + i], 0), rows) : rows;
      }
      if (i == 0) table.start = row0;
      base = uniform(value_of(sum, 63));
    }
  }
  __syncthreads();
}

// The tiles of a workgroup, one a round of the grid, up to kListTiles of them a launch: looked up by one thread each
// before their loop starts.  The search and its divisions inside the loop cost a microsecond a tile, and their registers
// spilled those of the 256 x 256 tiles.
//
// Each round is eight contiguous runs, one per XCD (workgroup b runs on XCD b mod 8), so that an XCD's L2 holds the rows
// and weights its tiles share; the last round's tiles are dealt to all XCDs alike.  A grid that eight does not divide
// takes every grid-th tile.
constexpr int kListTiles = 192;
struct TileList {
  GroupTile tile[kListTiles];  // e < 0: none
};

// Rounds from `round` on.  `order(tile, local)` places the group's local-th tile.  Every thread of the workgroup calls
// it; ends with a barrier.  SPLIT_BM: tiles of that many rows whose loop skips rows that are not there; where
// the last round has tiles for at most half or a quarter of the workgroups, a tile's rows go to two or four of them
// (`part`, and `m` as the end of the part's rows).
template <int SPLIT_BM = 0, class Order>
__device__ __forceinline__ void build_tile_list(TileList& list, const TileTable& table, int first, int groups, int round,
                                                Order&& order) {
  if (threadIdx.x < kListTiles) {  // workgroups have as many threads or more
    const uint32_t grid = gridDim.x, b = blockIdx.x;
    const int64_t base = ((int64_t)round + threadIdx.x) * grid, left = table.tiles[groups - 1] - base;
    const int64_t here = min((int64_t)grid, left);
    const uint32_t log_parts = SPLIT_BM == 0 || here < 0 ? 0 : here * 4 <= grid ? 2 : here * 2 <= grid ? 1 : 0;
    const uint32_t count = (uint32_t)here << log_parts, shift = grid & 7 ? 0 : 3, xcd = b & ((1u << shift) - 1);
    const uint32_t at = (xcd * count >> shift) + (b >> shift);
    GroupTile tile{-1, 0, 0, 0, 0, 0};
    if (left > 0 && at < ((xcd + 1) * count >> shift)) {
      const int t = (int)base + (int)(at >> log_parts);
      int lo = 0, hi = groups - 1;  // the first group with tiles[i] > t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (table.tiles[mid] > t) hi = mid;
        else lo = mid + 1;
      }
      const int row0 = lo ? table.ends[lo - 1] : table.start;
      tile = GroupTile{first + lo, row0, table.ends[lo] - row0, 0, 0, 0};  // a group with tiles has rows
      order(tile, t - (lo ? table.tiles[lo - 1] : 0));
      if (log_parts) {
        const int rows = SPLIT_BM >> log_parts;
        tile.part = (int)(at & ((1u << log_parts) - 1)) * rows;
        tile.m = min(tile.m, tile.tm * SPLIT_BM + tile.part + rows);
        if (tile.m <= tile.tm * SPLIT_BM + tile.part) tile.e = -1;  // the last round: nothing follows
      }
    }
    list.tile[threadIdx.x] = tile;
  }
  __syncthreads();
}

// The i-th tile of the list, wave-uniform; false past its end.
__device__ __forceinline__ bool listed_tile(const TileList& list, int i, GroupTile& g) {
  if (i >= kListTiles) return false;
  const GroupTile& x = list.tile[i];
  g = {uniform(x.e), uniform(x.row0), uniform(x.m), uniform(x.tm), uniform(x.tn), uniform(x.part)};
  return g.e >= 0;
}

__device__ __forceinline__ f32x16_t mfma_fp8(i32x8_t w, i32x8_t a, f32x16_t c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, a, c, 0, 0, 0, 0, 0, 0);
}

// The 8 e4m3 values of two dwords as bf16: exact, e4m3's range and 4 bits fit.
__device__ __forceinline__ bf16x8_t widen(int32_t lo, int32_t hi) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A lane's 32 bytes of a fragment, as they are (FAST) or widened.
template <bool FAST>
struct Fragment;
template <>
struct Fragment<true> {
  i32x8_t v;
  __device__ __forceinline__ void set(i32x8_t x) { v = x; }
};
template <>
struct Fragment<false> {
  bf16x8_t v[4];
  __device__ __forceinline__ void set(i32x8_t x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = widen(x[2 * i], x[2 * i + 1]);
  }
};
template <class ACC>
__device__ __forceinline__ ACC block_sum(const Fragment<true>& w, const Fragment<true>& a, ACC c) {
  return mfma_fp8(w.v, a.v, c);
}
template <class ACC>
__device__ __forceinline__ ACC block_sum(const Fragment<false>& w, const Fragment<false>& a, ACC c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(ACC) == 64)
      c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w.v[i], a.v[i], c, 0, 0, 0);
    else
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], a.v[i], c, 0, 0, 0);
  }
  return c;
}

__device__ __forceinline__ i32x8_t join(i32x4_t lo, i32x4_t hi) {
  return i32x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// The first `bytes` (any int) of a 16-byte chunk, zeros behind them.
__device__ __forceinline__ i32x4_t keep_bytes(i32x4_t v, int bytes) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int left = bytes - 4 * i;
    const uint32_t mask = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
    v[i] = (int32_t)((uint32_t)v[i] & mask);
  }
  return v;
}

// silu(g) * u as the definition has it; the e4m3 rounding behind it is far coarser than rcp's 1 ulp.
__device__ __forceinline__ float gated(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.0f + __expf(-g)) * u;
}

// max of |x| as bit patterns: a NaN is larger than everything else, so it reaches the scale.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// amax with its floor (as bits; positive floats order like their bits).
__device__ __forceinline__ float floored(uint32_t amax_bits) {
  return __builtin_bit_cast(float, max(amax_bits, __builtin_bit_cast(uint32_t, kAmaxFloor)));
}

__device__ __forceinline__ int32_t pack_e4m3(f32x4_t v) {
  int32_t r = 0;
  r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], r, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], r, true);
}

// One dword per lane by LDS-DMA: lane l's dword lands at `lds` + 4 l (see dma_copy16).
__device__ __forceinline__ void dma_copy4(u32x4_t rsrc, uint32_t voffset, uint32_t lds) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds"
               :
               : "v"(voffset), "s"(rsrc), "s"(lds)
               : "memory", "m0");
#pragma clang diagnostic pop
}

// E: the output type (EBf16, EF16, EF32) of a plain product.  GATED: w is [gate | up] of n = 2F rows,
// and a tile's BN weight rows are BN/2 = 128 gate rows and the 128 up rows that go with them.
template <class E, int BM_, int BN_, int WM_, int WN_, int STAGES_, bool GATED_, bool FAST_>
struct Fp8Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_;
  static constexpr bool GATED = GATED_, FAST = FAST_;
  using E16 = typename std::conditional<E::is_f32, EBf16, E>::type;  // 16-bit stores' type
  static constexpr int NW = WM * WN, NT = NW * 64;
  static constexpr int WTM = BM / WM, WTN = BN / WN, FM = WTM / 32, FN = WTN / 32;
  static constexpr int A_BYTES = BM * kScaleBlock, B_BYTES = BN * kScaleBlock;
  static constexpr int IA = A_BYTES / 1024, IB = B_BYTES / 1024;  // 1 KiB copies per stage: 8 rows of 128 bytes
  static constexpr int QA = IA / NW, QB = IB / NW;
  // Scales of a stage, in copies of 64 dwords: row scales, then the weight's, then unused ones.
  static constexpr int SA_COPIES = BM / 64;
  static constexpr int QS = (SA_COPIES + NW) / NW;  // copies a wave makes
  static constexpr int SCALE_BYTES = QS * NW * 256;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SCALE_BYTES;
  static constexpr int PER_STAGE = QA + QB + QS;  // copies of a wave per stage
  static constexpr int RED_BYTES = GATED ? BM * WN * 4 : 0;  // row maxima of the waves that share a row
  static constexpr int OUT_BYTES = GATED ? 0 : NW * 2048;    // 16 rows of a wave's columns on their way out
  static constexpr int TABLE_OFFSET = STAGES * STAGE_BYTES + RED_BYTES + OUT_BYTES;
  static constexpr int LDS_BYTES = TABLE_OFFSET + (int)(sizeof(TileTable) + sizeof(TileList));
  static constexpr int OUT_COLS = GATED ? BN / 2 : BN;  // output columns of a tile
  static_assert(IA % NW == 0 && IB % NW == 0, "every wave issues the same copies");
  static_assert(!GATED || (BN == 256 && FN == 2), "a gated tile is one 128-column block of the output");
  static_assert(LDS_BYTES <= 160 * 1024, "LDS of one CU");
  static_assert(STAGES * PER_STAGE < 64, "vmcnt is 6 bits");

  // What a wave's copies are made of: lane constants of the launch, and a tile's bases (wave-uniform).
  struct Copies {
    uint32_t a_off, b_off;     // first copy's byte offset in a panel; later ones are NW * 8 rows further on
    uint32_t a_step, b_step;   // NW * 8 rows in bytes
    uint32_t lds, lds_scale;
    int blocks;
    u32x4_t ra, rb, rb2;       // rb2: the up rows of a gated tile
    uint32_t s_off[QS];        // scale copies of this lane, or kOutOfRange
    const float* s_base[QS];
    int64_t s_step[QS];        // elements between blocks
  };

  __device__ static __forceinline__ void start(Copies& c, const Fp8Params& p, const char* smem) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    c.blocks = (p.k + kScaleBlock - 1) / kScaleBlock;
    c.lds = lds_address(smem) + (uint32_t)wave * 1024u;
    c.lds_scale = lds_address(smem) + (uint32_t)(A_BYTES + B_BYTES + wave * 256);
    // Row r of a panel keeps chunk c at c ^ swz_a(r, 8); wave w copies rows 8 (w + q NW) .. + 7.
    const int r0 = wave * 8 + lane / 8;
    const int ch = (lane & 7) ^ swz_a(r0, 8);  // swz_a of 8 chunks repeats every 32 rows, and NW * 8 is 32 or 64
    // The products stand apart from the sums: a 64-bit multiply-add would hold four registers over the loop.
    c.a_off = (uint32_t)r0 * (uint32_t)p.lda;
    c.b_off = (uint32_t)r0 * (uint32_t)p.ldw;
    asm volatile("" : "+v"(c.a_off), "+v"(c.b_off));
    c.a_off += (uint32_t)ch * 16u;
    c.b_off += (uint32_t)ch * 16u;
    asm volatile("" : "+v"(c.a_off), "+v"(c.b_off));
    c.a_step = (uint32_t)p.lda * (NW * 8);
    c.b_step = (uint32_t)p.ldw * (NW * 8);
  }

  __device__ static __forceinline__ void set_tile(Copies& c, const Fp8Params& p, const GroupTile& g, int wave) {
    const int tm = g.tm, tn = g.tn;
    const int lane = lane_here();
    const int m0 = tm * BM;
    const int valid_m = min(BM, g.m - m0);
    // A panel ends with the chunk that holds its last row's last k; what a copy reads past K inside it
    // (the next row's start) is cut in LDS.
    const uint32_t row_bytes = ((uint32_t)p.k + 15u) & ~15u;
    c.ra = make_rsrc(p.a + ((int64_t)g.row0 + m0) * p.lda, (uint32_t)(valid_m - 1) * (uint32_t)p.lda + row_bytes);
    const uint8_t* w = p.w + (int64_t)g.e * p.swg;
    const int f = p.n >> 1;
    const int n0 = tn * OUT_COLS;
    const int valid_n = GATED ? min(BN / 2, f - n0) : min(BN, p.n - n0);
    const uint32_t b_bytes = (uint32_t)(valid_n - 1) * (uint32_t)p.ldw + row_bytes;
    c.rb = make_rsrc(w + (int64_t)n0 * p.ldw, b_bytes);
    if constexpr (GATED) c.rb2 = make_rsrc(w + (int64_t)(f + n0) * p.ldw, b_bytes);
    // Scales: copy j < SA_COPIES fetches the scales of rows 64 j .. + 63, the next one the weight's.  Plain: lane i
    // has the tile's weight rows from 128 i on.  Gated: lanes 0 to 15 have eight up rows each (up rows start at any
    // multiple of 8, so a scale block may end between any two of them), lane 16 the gate rows.
    const int last = (p.n + kScaleBlock - 1) / kScaleBlock - 1;
    const int block = GATED && lane < 16 ? (f + n0 + 8 * lane) / kScaleBlock : n0 / kScaleBlock + (GATED ? 0 : lane);
    const uint32_t w_off = lane < (GATED ? 17 : 4) ? (uint32_t)min(block, last) * (uint32_t)p.ssn * 4u : kOutOfRange;
#pragma unroll
    for (int q = 0; q < QS; ++q) {
      const int j = wave + q * NW, row = j * 64 + lane;
      const bool rows = j < SA_COPIES;
      c.s_base[q] = uniform(rows ? p.sa + ((int64_t)g.row0 + m0) * p.sam : p.sw + (int64_t)g.e * p.ssg);
      c.s_step[q] = uniform(rows ? p.sak : p.ssk);
      if (rows) c.s_off[q] = row < valid_m ? (uint32_t)row * (uint32_t)p.sam * 4u : kOutOfRange;
      else c.s_off[q] = j == SA_COPIES ? w_off : kOutOfRange;
    }
  }

  // Copies of a slice are spread over the steps in which its buffer is free: the FN steps after the barrier of the
  // slice that held it and the first EARLY steps of the next one, weights (which come from HBM) first.  Issued
  // in one burst they kept every wave from its matrix instructions until the last was accepted.
  static constexpr int BEFORE = (FM - 1) * FN;  // steps before a slice's barrier: every read of it is under way
  static constexpr int EARLY = FM * FN >= 8 ? 3 : 0;
  static constexpr int PARTS = FN + EARLY;
  static constexpr int first_copy(int part) { return (part * PER_STAGE + PARTS - 1) / PARTS; }

  // Part [PART0, PART1) of slice kt's copies.
  template <int PART0, int PART1>
  __device__ static __forceinline__ void issue(const Copies& c, int stage, int kt) {
    const uint32_t base = c.lds + (uint32_t)(stage * STAGE_BYTES);
    uint32_t k0 = (uint32_t)kt * kScaleBlock;
    asm volatile("" : "+s"(k0));  // no running sums of it and the offsets in vector registers
    uint32_t a0 = c.a_off + k0, b0 = c.b_off + k0;
    // The steps are added here: hoisted out of the loop, the offsets of eight copies took spilled registers.
    asm volatile("" : "+v"(a0), "+v"(b0));
#pragma unroll
    for (int i = first_copy(PART0); i < first_copy(PART1); ++i) {
      if (i < QB) {
        const bool up = GATED && i >= QB / 2;
        dma_copy16(up ? c.rb2 : c.rb, b0 + (uint32_t)(up ? i - QB / 2 : i) * c.b_step,
                   base + (uint32_t)(A_BYTES + i * NW * 1024));
      } else if (i < QB + QA) {
        const int q = i - QB;
        dma_copy16(c.ra, a0 + (uint32_t)q * c.a_step, base + (uint32_t)(q * NW * 1024));
      } else {
        const int q = i - QB - QA;
        dma_copy4(make_rsrc(c.s_base[q] + min(kt, c.blocks - 1) * c.s_step[q], kOutOfRange), c.s_off[q],
                  c.lds_scale + (uint32_t)(stage * STAGE_BYTES + q * NW * 256));
      }
    }
  }

  // This lane's first 16-byte chunk in the 32 rows of a fragment: every panel row group of 32 has the same
  // swizzle, so one offset serves both panels, and the lane's other three chunks of the row differ from it
  // in bits 5 and 6 only.
  __device__ static __forceinline__ uint32_t lane_offset() {
    const int lane = threadIdx.x & 63, row = lane & 31;
    return (uint32_t)(row * kScaleBlock + (((lane >> 5) ^ swz_a(row, 8)) << 4));
  }
  // LDS addresses of the four chunks in the row group that starts `rows` bytes into LDS (a multiple of 128).
  struct Chunks {
    uint32_t at[4];
  };
  __device__ static __forceinline__ Chunks chunks(uint32_t lane, uint32_t rows) {
    Chunks c;
    c.at[0] = rows + lane;
#pragma unroll
    for (int i = 1; i < 4; ++i) c.at[i] = c.at[0] ^ (uint32_t)(i << 5);
    return c;
  }

  // 32 bytes of a panel row for the j-th 64-byte half of the slice, `rows32` row groups on.
  __device__ static __forceinline__ i32x8_t frag(const char* smem, const Chunks& c, int rows32, int j) {
    const char* p = smem + rows32 * 32 * kScaleBlock;
    return join(*reinterpret_cast<const i32x4_t*>(p + c.at[2 * j]),
                *reinterpret_cast<const i32x4_t*>(p + c.at[2 * j + 1]));
  }

  // Zeros to the bytes of a landed slice from `left` (< 128, any sign) on: a K that is no multiple of 128
  // ends inside it.  A thread per panel row.
  __device__ static __forceinline__ void cut_tail(char* stage, int left, int wave) {
    for (int r = wave * 64 + lane_here(); r < BM + BN; r += NT) {
      // Panel rows of A, then of B, are 128 bytes each; swz_a repeats every 32 rows and BM is a multiple of it.
      for (int c = max(left, 0) >> 4; c < 8; ++c) {
        i32x4_t* chunk = reinterpret_cast<i32x4_t*>(stage + r * kScaleBlock + ((c ^ swz_a(r, 8)) << 4));
        *chunk = keep_bytes(*chunk, left - c * 16);
      }
    }
  }

  // First panel row of a wave's columns: gated waves hold their gate rows' fragments, then the up rows',
  // which lie BN / 2 rows after the gate rows.
  __device__ static __forceinline__ int b_row(int wave_n) { return wave_n * (GATED ? WTN / 2 : WTN); }

  // What a wave holds of the slice it works on.  a is double-buffered over row fragments; the first
  // fragments of the next slice replace these while the last ones are multiplied.
  struct Slice {
    Fragment<FAST> a[2][2], b[FN][2];
    float sa[2];
    float sw[GATED ? 5 : 1];  // wave-uniform; gated: of each eight up rows of the wave's 32, then the gate's
  };
  // `a`: the chunks of the wave's first row group of the slice; `lane` lane_offset(); `stage` the slice's LDS offset.
  __device__ static __forceinline__ void load_a(Slice& s, const char* smem, const Chunks& a, uint32_t lane, uint32_t stage,
                                                int wave_m, int fm) {
#pragma unroll
    for (int j = 0; j < 2; ++j) s.a[fm & 1][j].set(frag(smem, a, fm, j));
    s.sa[fm & 1] = *reinterpret_cast<const float*>(smem + stage + A_BYTES + B_BYTES + (wave_m * WTM + fm * 32) * 4 +
                                                   ((lane / (kScaleBlock / 4)) & 124));  // 4 (lane's row)
  }
  __device__ static __forceinline__ void load_b(Slice& s, const char* smem, const Chunks& b, int fn) {
    constexpr int UP = GATED ? (BN / 2 - WTN / 2) / 32 : 0;  // row groups from a wave's gate rows' end to its up rows
#pragma unroll
    for (int j = 0; j < 2; ++j) s.b[fn][j].set(frag(smem, b, fn + (GATED && fn >= FN / 2 ? UP : 0), j));
  }
  __device__ static __forceinline__ void load_weight_scales(Slice& s, const char* smem, uint32_t stage, int wave_n) {
    const float* sw = reinterpret_cast<const float*>(smem + stage + A_BYTES + B_BYTES) + SA_COPIES * 64;
    if constexpr (GATED) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s.sw[i] = uniform(sw[wave_n * (WTN / 16) + i]);
      s.sw[4] = uniform(sw[16]);
    } else {
      static_assert(kScaleBlock % WTN == 0, "a wave's columns lie in one scale block");
      s.sw[0] = uniform(sw[wave_n * WTN / kScaleBlock]);
    }
  }

  // A fragment's sum of one block, waiting to be added while the next one's is formed.
  struct Pending {
    f32x16_t t;
    float s;     // the sum's scale; up rows of a gated tile: the row scale alone, and
    float w[4];  // the weight's (wave-uniform) for each quad of registers, eight up rows
  };
  // acc += t * scale for B fragment fn.
  __device__ static __forceinline__ void add(f32x16_t& acc, const Pending& p, int fn) {
    if (GATED && fn >= FN / 2) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float s = p.s * p.w[q];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[q * 4 + i] += p.t[q * 4 + i] * s;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] += p.t[i] * p.s;
    }
  }

  // Steps [X0, X1) of a slice: step x forms fragment (x / FN, x % FN)'s block sum and adds the one before.
  // The last sum of a slice is added in the next one.  `copies(part)` issues a part of a slice's copies.
  template <int X0, int X1, class Issue>
  __device__ static __forceinline__ void steps(f32x16_t (&acc)[FM][FN], Slice& s, Pending (&pend)[2], const char* smem,
                                               const Chunks& a, uint32_t lane, uint32_t stage, Issue&& copies,
                                               int wave_m) {
    unroll_steps<X0, X1>([&](auto step) {
      constexpr int x = decltype(step)::value;
      constexpr int fm = x / FN, fn = x % FN, last = x == 0 ? FM * FN - 1 : x - 1;
      constexpr int part = x >= BEFORE ? x - BEFORE : x < EARLY ? FN + x : -1;
      if constexpr (part >= 0) copies(std::integral_constant<int, part>{});
      if (fn == 0 && fm + 1 < FM) load_a(s, smem, a, lane, stage, wave_m, fm + 1);
      Pending& p = pend[x & 1];
      p.t = f32x16_t{};
#pragma unroll
      for (int j = 0; j < 2; ++j) p.t = block_sum(s.b[fn][j], s.a[fm & 1][j], p.t);
      if constexpr (GATED && fn >= FN / 2) {
        p.s = s.sa[fm & 1];
#pragma unroll
        for (int q = 0; q < 4; ++q) p.w[q] = s.sw[q];
      } else {
        p.s = s.sa[fm & 1] * s.sw[GATED ? 4 : 0];
      }
      f32x16_t& to = acc[last / FN][last % FN];
      add(to, pend[(x + 1) & 1], last % FN);
      // The sum is made here and now: put off past the slice's barrier, every pending sum would stay alive.
      asm volatile("" : "+v"(to));
      if constexpr (FAST) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 9, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 9, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    });
  }
  template <int X0, int X1, class F>
  __device__ static __forceinline__ void unroll_steps(F&& f) {
    if constexpr (X0 < X1) {
      f(std::integral_constant<int, X0>{});
      unroll_steps<X0 + 1, X1>(f);
    }
  }
  static_assert((FM * FN) % 2 == 0 && FM % 2 == 0, "pending sums and row fragments alternate");

  __device__ static __forceinline__ void store_plain(const f32x16_t (&acc)[FM][FN], const Fp8Params& p,
                                                     const GroupTile& g, char* smem, int wave_m, int wave_n) {
    const int lane = lane_here(), tm = g.tm, tn = g.tn;
    constexpr int ES = sizeof(typename E::raw);
    const int m0 = tm * BM, n0 = tn * BN;
    char* base = static_cast<char*>(p.out) + (((int64_t)g.row0 + m0) * p.ldo + n0) * ES;
    const int valid_m = min(BM, g.m - m0), valid_n = p.n - n0;
    if (ES == 2 && p.n % 8 == 0 && p.ldo % 8 == 0 && p.ldo < (1 << 22) && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0) {
      // Through LDS, 16 rows of the wave's 64 columns at a time (16-byte chunk c of row r at c ^ r), so that a store
      // covers whole 128-byte lines: from the registers, 32 bytes of a row at a time, 16384 rows of [7168, 2048] x 32
      // took 269 us instead of 252.  Non-temporal, so that the operands keep the L2: 128x256 tiles 339 -> 324 us there, the
      // others unchanged.  One buffer resource ends with the tile's last valid row.
      static_assert(WTN == 64, "a wave's 16-bit rows are 128 bytes");
      const uint32_t pitch = (uint32_t)p.ldo * ES;
      const auto rs = __builtin_amdgcn_make_buffer_rsrc(
          base, (short)0, (int)((uint32_t)(valid_m - 1) * pitch + (uint32_t)valid_n * ES), (int)kBufferFlags);
      char* slot = smem + STAGES * STAGE_BYTES + (wave_m * WN + wave_n) * 2048;
      const int r = lane & 15, col = wave_n * WTN + (lane & 7) * 8;
#pragma unroll
      for (int fm = 0; fm < FM; ++fm)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (((lane >> 4) & 1) == half) {
#pragma unroll
            for (int fn = 0; fn < FN; ++fn)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const f32x16_t& v = acc[fm][fn];
                *reinterpret_cast<u32x2_t*>(slot + r * 128 + (((fn * 4 + q) ^ (r & 7)) << 4) + (lane >> 5) * 8) =
                    pack4<E16>(f32x4_t{v[q * 4], v[q * 4 + 1], v[q * 4 + 2], v[q * 4 + 3]});
              }
          }
          compiler_fence();
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int at = j * 8 + (lane >> 3), row = wave_m * WTM + fm * 32 + half * 16 + at;
            const u32x4_t x = *reinterpret_cast<const u32x4_t*>(slot + at * 128 + (((lane & 7) ^ (at & 7)) << 4));
            __builtin_amdgcn_raw_buffer_store_b128(
                x, rs, col < valid_n ? (uint32_t)row * pitch + (uint32_t)col * ES : kOutOfRange, 0, kNonTemporal);
          }
          compiler_fence();
        }
      return;
    }
    const bool vec = p.n % 4 == 0 && p.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & (4 * ES - 1)) == 0;
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      const int row = wave_m * WTM + fm * 32 + (lane & 31);
      char* out = base + (int64_t)row * p.ldo * ES;
      if (row >= valid_m) continue;
#pragma unroll
      for (int fn = 0; fn < FN; ++fn)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = wave_n * WTN + fn * 32 + q * 8 + (lane >> 5) * 4;
          const f32x4_t v = {acc[fm][fn][q * 4], acc[fm][fn][q * 4 + 1], acc[fm][fn][q * 4 + 2],
                             acc[fm][fn][q * 4 + 3]};
          if (vec) {
            if (n < valid_n) store4<E>(out + (int64_t)n * ES, v);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (n + i < valid_n) store1<E>(out + (int64_t)(n + i) * ES, v[i]);
          }
        }
    }
  }

  // silu(gate) * up of the tile's 128 output columns, their maximum per row over the waves that share
  // it (through `red`), and the quantised row.
  __device__ static __forceinline__ void store_gated(f32x16_t (&acc)[FM][FN], const Fp8Params& p, const GroupTile& g,
                                                     int tm, int tn, int wave_m, int wave_n, uint32_t* red) {
    const int lane = lane_here();
    const int f = p.n >> 1;
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      uint32_t top = 0;
#pragma unroll
      for (int fn = 0; fn < FN / 2; ++fn)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float h = gated(acc[fm][fn][i], acc[fm][fn + FN / 2][i]);
          acc[fm][fn][i] = h;
          top = max(top, abs_bits(h));  // columns past F are zeros
        }
      const auto other = __builtin_amdgcn_permlane32_swap(top, top, false, false);
      top = max(other[0], other[1]);
      if (lane < 32) red[(wave_m * WTM + fm * 32 + lane) * WN + wave_n] = top;
    }
    __syncthreads();
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      const int local = wave_m * WTM + fm * 32 + (lane & 31);
      const int row = tm * BM + local;
      uint32_t top = 0;
#pragma unroll
      for (int w = 0; w < WN; ++w) top = max(top, red[local * WN + w]);
      const float amax = floored(top);
      const float inverse = kE4m3Max / amax;
      const bool in_m = row < g.m;
      if (in_m && wave_n == 0 && lane < 32)
        p.out_scale[((int64_t)g.row0 + row) * p.osm + (int64_t)tn * p.osk] = amax / kE4m3Max;
      uint8_t* out = static_cast<uint8_t*>(p.out) + ((int64_t)g.row0 + row) * p.ldo;
#pragma unroll
      for (int fn = 0; fn < FN / 2; ++fn)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          f32x4_t v, u;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[i] = acc[fm][fn][q * 4 + i] * inverse;
            u[i] = acc[fm][fn][q * 4 + 4 + i] * inverse;
          }
          const auto s = __builtin_amdgcn_permlane32_swap(pack_e4m3(v), pack_e4m3(u), false, false);
          const int n = tn * (BN / 2) + wave_n * (WTN / 2) + fn * 32 + q * 8 + (lane >> 5) * 8;
          if (in_m && n < f) *MOEGEMM_GLOBAL(u32x2_t, out + n) = u32x2_t{s[0], s[1]};
        }
    }
  }
};

// Prefill tiles.  Bound by the matrix instructions and what keeps them waiting: 50 to 57 % of the time they are busy
// (16384 rows over 32 experts), the rest goes to the scaled additions (without them 9 % less time), the LDS copies and
// the barrier of each slice.  256x256 tiles, 8 waves: the widest that two 64 KiB buffers and 256 registers a lane allow,
// so each operand byte is copied to LDS least often.  Fast sums: 8192^3 458 us, 2.40 PFLOP/s; 16384 rows of 32 x
// [7168, 2048] 252 us, 1.91 PFLOP/s; of 32 x [4096, 7168] with the gated epilogue 477 us, 2.02 PFLOP/s.  Exact sums
// hold 128x256 outputs at most (widened fragments take the registers): 455 us, 1.06 PFLOP/s of the 1.69 that the bf16
// instruction alone reaches.
//
// The slices of a workgroup's tiles form one stream: while slice i is multiplied, slice i + 1 has landed
// or is about to, and its first fragments are read under slice i's last matrix instructions.  There is one barrier
// per slice, before its last row of fragments, when every wave has read all of the slice: behind it the
// slice's buffer takes slice i + 2, of this tile or the next, so a tile's end does not drain the pipeline.
template <class T>
__global__ void __launch_bounds__(T::NT) fp8_tile_kernel(Fp8Params p) {
  static_assert(T::STAGES == 2, "two buffers: slice i + 2 takes slice i's");
  __shared__ __attribute__((aligned(16))) char smem[T::LDS_BYTES];
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wave_m = wave / T::WN, wave_n = wave % T::WN;
  const int blocks = (p.k + kScaleBlock - 1) / kScaleBlock;
  const int kt_count = max(blocks, 2);
  const bool cut = p.k % kScaleBlock != 0;  // slices from K / 128 on are cut in LDS
  TileTable& table = *reinterpret_cast<TileTable*>(smem + T::TABLE_OFFSET);
  TileList& list = *reinterpret_cast<TileList*>(smem + T::TABLE_OFFSET + sizeof(TileTable));
  build_tile_table(table, p.offs, p.first, p.groups, p.rows, T::BM, p.n_tiles);
  build_tile_list(list, table, p.first, p.groups, p.round, [&](GroupTile& tile, int local) {
    group_m_order(local, (tile.m + T::BM - 1) / T::BM, p.n_tiles, 8, tile.tm, tile.tn);
  });
  GroupTile g;
  if (!listed_tile(list, 0, g)) return;
  typename T::Copies c;
  T::start(c, p, smem);
  T::set_tile(c, p, g, wave);
  T::template issue<0, T::PARTS>(c, 0, 0);
  T::template issue<0, T::FN>(c, 1, 1);  // the rest of it under slice 0's first steps
  wait_vmcnt<T::first_copy(T::FN)>();
  __builtin_amdgcn_s_barrier();
  compiler_fence();
  if (cut && blocks == 1) {
    T::cut_tail(smem, p.k, wave);
    __syncthreads();
  }
  const uint32_t lane = T::lane_offset();
  typename T::Slice s;
  typename T::Chunks ca;
  auto load_first = [&](uint32_t stage) {
    T::load_weight_scales(s, smem, stage, wave_n);
    ca = T::chunks(lane, stage + (uint32_t)(wave_m * T::WTM * kScaleBlock));
    T::load_a(s, smem, ca, lane, stage, wave_m, 0);
    const typename T::Chunks cb = T::chunks(lane, stage + (uint32_t)(T::A_BYTES + T::b_row(wave_n) * kScaleBlock));
#pragma unroll
    for (int fn = 0; fn < T::FN; ++fn) T::load_b(s, smem, cb, fn);
  };
  load_first(0);

  int buffer = 0, i = 0;
  bool more = true;
  while (more) {
    f32x16_t acc[T::FM][T::FN];
#pragma unroll
    for (int fm = 0; fm < T::FM; ++fm)
#pragma unroll
      for (int fn = 0; fn < T::FN; ++fn) acc[fm][fn] = f32x16_t{};
    typename T::Pending pend[2] = {};
    // One slice.  `early(part)` issues the rest of slice i + 1's copies into the other buffer, `late(part)`
    // the first of slice i + 2's into this one; `left()` says how many bytes of the next slice's rows lie inside K.
    auto slice = [&](auto&& early, auto&& late, auto&& left) {
      const uint32_t cur = (uint32_t)(buffer * T::STAGE_BYTES), next = (uint32_t)((buffer ^ 1) * T::STAGE_BYTES);
      T::template steps<0, T::BEFORE>(acc, s, pend, smem, ca, lane, cur, early, wave_m);
      // Every fragment of this slice is in registers, and the next slice has landed.
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      compiler_fence();
      if (const int bytes = left(); bytes < kScaleBlock) {
        T::cut_tail(smem + next, bytes, wave);
        __syncthreads();
      }
      // Fragments of the next slice (of the next tile, behind the last one) as this one's fall free.
      T::template steps<T::BEFORE, T::FM * T::FN>(acc, s, pend, smem, ca, lane, cur, late, wave_m);
      load_first(next);
      buffer ^= 1;
    };
    auto issue = [&](auto part, int stage, int kt) {
      T::template issue<decltype(part)::value, decltype(part)::value + 1>(c, stage, kt);
    };
    // The loop is kept free of branches: the copies are issued between matrix instructions.
    for (int kt = 0; kt + 2 < kt_count; ++kt)
      slice([&](auto part) { issue(part, buffer ^ 1, kt + 1); }, [&](auto part) { issue(part, buffer, kt + 2); },
            [] { return kScaleBlock; });
    // The last two slices refill with the next tile's first two.
    GroupTile g_next{};
    more = listed_tile(list, ++i, g_next);
    for (int ahead = 0; ahead < 2; ++ahead)
      slice([&](auto part) { if (ahead == 0 || more) issue(part, buffer ^ 1, ahead == 0 ? kt_count - 1 : 0); },
            [&](auto part) { if (more) issue(part, buffer, ahead); },
            [&] {
              if (ahead == 0 && more) T::set_tile(c, p, g_next, wave);
              return p.k - (ahead == 0 ? kt_count - 1 : 0) * kScaleBlock;
            });
    T::add(acc[T::FM - 1][T::FN - 1], pend[(T::FM * T::FN - 1) & 1], T::FN - 1);
    if constexpr (T::GATED)
      T::store_gated(acc, p, g, g.tm, g.tn, wave_m, wave_n,
                     reinterpret_cast<uint32_t*>(smem + T::STAGES * T::STAGE_BYTES));
    else
      T::store_plain(acc, p, g, smem, wave_m, wave_n);
    g = g_next;
  }
}

// Decode: 16 FM rows of a group by 16 FN weight rows per wave, WN waves along the columns, WK waves that take
// the K blocks wk, wk + WK, ...  Bound by HBM where a group's rows fit a unit: each weight byte is then read once.  A
// group of more rows is walked by the same workgroups, 16 FM rows at a time, and its weights are read again each time.
//
// Every wave streams on its own: a ring of STAGES slots in LDS, one K block of its weights, rows and scales each,
// filled by DMA in whole 128-byte lines and refilled as soon as its fragments are in registers.  No barrier
// and no wait of other waves is involved, and the ring runs on over the units (group, column tile, row tile) of the
// workgroup, so nothing drains between them.  Loads of fragments straight into registers read half lines:
// 256 rows over 32 experts of [4096, 7168] took 171 to 197 us that way whatever the tile and depth, and 142 us (6.6
// TB/s) this way.
template <class E, int FM_, int FN_, int WN_, int WK_, int STAGES_, bool GATED_>
struct Fp8Stream {
  static constexpr int FM = FM_, FN = FN_, WN = WN_, WK = WK_, STAGES = STAGES_;
  static constexpr bool GATED = GATED_;
  static constexpr int NW = WN * WK, NT = NW * 64;
  static constexpr int BM = 16 * FM, BN = 16 * FN * WN;
  static constexpr int OUT_COLS = GATED ? BN / 2 : BN;
  static constexpr int FRAGS = FM * FN * WN;  // accumulator fragments of a tile
  static constexpr int W_BYTES = FN * 16 * kScaleBlock, A_BYTES = FM * 16 * kScaleBlock;
  static constexpr int SLOT_BYTES = W_BYTES + A_BYTES + 512;  // and two copies of scales: rows, weights
  static constexpr int COPIES = 2 * FN + 2 * FM + 2;
  static constexpr int RING_BYTES = NW * STAGES * SLOT_BYTES;
  static constexpr int RED_BYTES = WK > 1 ? WK * FRAGS * 1024 : 0;
  static constexpr int LDS_BYTES = RING_BYTES + RED_BYTES + (GATED ? BM * 8 * 4 : 0);
  static_assert(kScaleBlock % (16 * FN) == 0, "a wave's columns lie in one scale block");
  static_assert(!GATED || (OUT_COLS == kScaleBlock && FN == 4 && WK == 1), "a gated tile is one block of the output");
  static_assert(LDS_BYTES <= 160 * 1024, "LDS of one CU");
  static_assert(STAGES * COPIES < 64, "vmcnt is 6 bits");
};

template <class T, class E>
__global__ void __launch_bounds__(T::NT) fp8_stream_kernel(Fp8Params p) {
  constexpr int FM = T::FM, FN = T::FN, WN = T::WN, WK = T::WK, STAGES = T::STAGES;
  constexpr bool GATED = T::GATED;
  __shared__ __attribute__((aligned(16))) char smem[T::LDS_BYTES];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wn = wave % WN, wk = wave / WN;
  const int f = p.n >> 1;
  const int blocks = (p.k + kScaleBlock - 1) / kScaleBlock;
  const int rounds = (blocks + WK - 1) / WK;  // K blocks of every wave; those past the end are zeros
  const int units = p.groups * p.n_tiles;
  const int last_n = (p.n + kScaleBlock - 1) / kScaleBlock - 1;

  // A place in the workgroup's stream of (unit, row tile, K block).
  struct Cursor {
    int unit, e, tn, row0, m, m0, round;
  };
  auto find_rows = [&](Cursor& c) {  // the first unit from c.unit on whose group has rows
    for (; c.unit < units; c.unit += gridDim.x) {
      c.e = c.unit / p.n_tiles;
      c.tn = c.unit - c.e * p.n_tiles;
      c.row0 = group_rows(p.offs, p.rows, c.e, c.m);
      if (c.m > 0) break;
    }
    c.m0 = 0;
    c.round = 0;
  };
  auto advance = [&](Cursor& c) {  // true at a new unit or row tile
    if (++c.round < rounds) return false;
    c.round = 0;
    c.m0 += T::BM;
    if (c.m0 < c.m) return true;
    c.unit += gridDim.x;
    find_rows(c);
    return true;
  };

  // Copies: eight rows of 128 bytes each.  Chunk c of row r lies at c ^ (r / 2 % 8), which puts the 16 rows a
  // fragment reads at one chunk on all banks; two copies further on it is the same, next door it differs in bit 2.
  const uint32_t ring = (uint32_t)(wave * STAGES * T::SLOT_BYTES);
  const uint32_t ring_lds = lds_address(smem) + ring;
  const uint32_t row_bytes = ((uint32_t)p.k + 15u) & ~15u;
  const uint32_t copy_chunk = (uint32_t)((lane & 7) ^ (lane >> 4)) * 16u;
  const uint32_t w_row = (uint32_t)(lane >> 3) * (uint32_t)p.ldw, a_row = (uint32_t)(lane >> 3) * (uint32_t)p.lda;
  const uint32_t w_even = w_row + copy_chunk, w_odd = w_row + (copy_chunk ^ 64u);
  const uint32_t a_even = a_row + copy_chunk, a_odd = a_row + (copy_chunk ^ 64u);
  // What a unit's copies are made of.  A panel ends with the chunk that holds its last row's last k; what a copy
  // reads past K inside it is cut from the fragments.
  u32x4_t rw, rw2, ra, rs, rt;
  uint32_t rw_bytes = 0, ra_bytes = 0, s_off = 0, t_off = 0;
  const float *s_base = nullptr, *t_base = nullptr;
  auto set_unit = [&](const Cursor& c) {
    const int n0 = c.tn * T::OUT_COLS + wn * (GATED ? 8 : 16) * FN;
    const int valid_m = min(T::BM, c.m - c.m0);
    const int valid_n = min(GATED ? f - n0 : p.n - n0, GATED ? 8 * FN : 16 * FN);
    const uint8_t* w = p.w + (int64_t)c.e * p.swg + (int64_t)n0 * p.ldw;
    rw_bytes = valid_n > 0 ? (uint32_t)(valid_n - 1) * (uint32_t)p.ldw + row_bytes : 0;
    ra_bytes = (uint32_t)(valid_m - 1) * (uint32_t)p.lda + row_bytes;
    rw = make_rsrc(w, rw_bytes);
    if constexpr (GATED) rw2 = make_rsrc(w + (int64_t)f * p.ldw, rw_bytes);
    ra = make_rsrc(p.a + ((int64_t)c.row0 + c.m0) * p.lda, ra_bytes);
    s_base = p.sa + ((int64_t)c.row0 + c.m0) * p.sam + (int64_t)wk * p.sak;
    s_off = lane < valid_m ? (uint32_t)lane * (uint32_t)p.sam * 4u : kOutOfRange;
    // The weight's scales: one block for the wave's columns; gated: lanes 0 to 3 eight up rows each, lane 4 the gate's.
    const int block = min((GATED && lane < 4 ? f + n0 + 8 * lane : n0) / kScaleBlock, last_n);
    t_base = p.sw + (int64_t)c.e * p.ssg + (int64_t)wk * p.ssk;
    t_off = lane < 5 ? (uint32_t)block * (uint32_t)p.ssn * 4u : kOutOfRange;
  };
  auto issue = [&](const Cursor& c, int slot) {
    const uint32_t to = ring_lds + (uint32_t)(slot * T::SLOT_BYTES);
    const int kb = wk + c.round * WK;
    const uint32_t k0 = (uint32_t)kb * kScaleBlock;
    const bool in = kb < blocks;  // else zeros: values, and scales of either side
    rw[2] = in ? rw_bytes : 0;
    if constexpr (GATED) rw2[2] = rw[2];
    ra[2] = in ? ra_bytes : 0;
    uint32_t w0 = w_even + k0, w1 = w_odd + k0, a0 = a_even + k0, a1 = a_odd + k0;
    asm volatile("" : "+v"(w0), "+v"(w1), "+v"(a0), "+v"(a1));  // the rows' steps are added here
#pragma unroll
    for (int q = 0; q < 2 * FN; ++q) {
      const bool up = GATED && q >= FN;
      dma_copy16_nt(up ? rw2 : rw, (q & 1 ? w1 : w0) + (uint32_t)((up ? q - FN : q) * 8) * (uint32_t)p.ldw,
                 to + (uint32_t)(q * 1024));
    }
#pragma unroll
    for (int q = 0; q < 2 * FM; ++q)
      dma_copy16(ra, (q & 1 ? a1 : a0) + (uint32_t)(q * 8) * (uint32_t)p.lda, to + (uint32_t)(T::W_BYTES + q * 1024));
    rs = make_rsrc(s_base + (int64_t)c.round * WK * p.sak, in ? kOutOfRange : 0);
    dma_copy4(rs, s_off, to + (uint32_t)(T::W_BYTES + T::A_BYTES));
    rt = make_rsrc(t_base + (int64_t)c.round * WK * p.ssk, in ? kOutOfRange : 0);
    dma_copy4(rt, t_off, to + (uint32_t)(T::W_BYTES + T::A_BYTES + 256));
  };

  Cursor next{(int)blockIdx.x, 0, 0, 0, 0, 0, 0};
  find_rows(next);
  if (next.unit >= units) return;
  Cursor at = next;
  set_unit(next);
  for (int s = 0; s < STAGES; ++s) {
    if (next.unit >= units) break;
    issue(next, s);
    if (advance(next) && next.unit < units) set_unit(next);
  }

  // This lane's chunks of a fragment: row lane % 16, chunks lane / 16 and 4 + lane / 16.
  const int frag_row = lane & 15, group = lane >> 4;
  const uint32_t frag_lo = (uint32_t)(frag_row * kScaleBlock + ((group ^ (frag_row >> 1)) << 4)), frag_hi = frag_lo ^ 64u;
  auto frag = [&](const char* rows, int i, int left) {
    i32x4_t lo = *reinterpret_cast<const i32x4_t*>(rows + i * 16 * kScaleBlock + frag_lo);
    i32x4_t hi = *reinterpret_cast<const i32x4_t*>(rows + i * 16 * kScaleBlock + frag_hi);
    if (left < kScaleBlock) {  // K ends inside the block
      lo = keep_bytes(lo, left - group * 16);
      hi = keep_bytes(hi, left - 64 - group * 16);
    }
    return join(lo, hi);
  };

  f32x4_t acc[FM][FN];
#pragma unroll
  for (int fm = 0; fm < FM; ++fm)
#pragma unroll
    for (int fn = 0; fn < FN; ++fn) acc[fm][fn] = f32x4_t{};

  for (int slot = 0; at.unit < units; slot = slot + 1 == STAGES ? 0 : slot + 1) {
    // The slot has landed once only the younger ones' copies are outstanding (near the end there are fewer).
    if (next.unit < units) wait_vmcnt<(STAGES - 1) * T::COPIES>();
    else wait_vmcnt<0>();
    compiler_fence();
    const char* from = smem + ring + slot * T::SLOT_BYTES;
    const int left = p.k - (wk + at.round * WK) * kScaleBlock;
    i32x8_t av[FM], wv[FN];
    float sa[FM], sw[FN];
#pragma unroll
    for (int fn = 0; fn < FN; ++fn) wv[fn] = frag(from, fn, left);
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      av[fm] = frag(from + T::W_BYTES, fm, left);
      sa[fm] = reinterpret_cast<const float*>(from + T::W_BYTES + T::A_BYTES)[fm * 16 + frag_row];
    }
    const float* scales = reinterpret_cast<const float*>(from + T::W_BYTES + T::A_BYTES + 256);
#pragma unroll
    for (int fn = 0; fn < FN; ++fn)
      // A lane's four columns of an up fragment lie in one eight.
      sw[fn] = scales[!GATED ? 0 : fn < FN / 2 ? 4 : (fn - FN / 2) * 2 + (group >> 1)];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (next.unit < units) {
      issue(next, slot);
      if (advance(next) && next.unit < units) set_unit(next);
    }
    Fragment<false> a[FM];
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) a[fm].set(av[fm]);
#pragma unroll
    for (int fn = 0; fn < FN; ++fn) {
      Fragment<false> b;
      b.set(wv[fn]);
#pragma unroll
      for (int fm = 0; fm < FM; ++fm) {
        const f32x4_t t = block_sum(b, a[fm], f32x4_t{});
        const float s = sa[fm] * sw[fn];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[fm][fn][i] += t[i] * s;
      }
    }
    if (at.round + 1 < rounds) {
      ++at.round;
      continue;
    }

    const int valid_m = min(T::BM, at.m - at.m0);
    const int64_t first = (int64_t)at.row0 + at.m0;
    if constexpr (!GATED) {
      constexpr int ES = sizeof(typename E::raw);
      const bool vec = p.n % 4 == 0 && p.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & (4 * ES - 1)) == 0;
      auto store = [&](const f32x4_t& v, int fm, int fn, int fw) {
        const int row = fm * 16 + frag_row;
        const int n = at.tn * T::BN + fw * 16 * FN + fn * 16 + group * 4;
        if (row >= valid_m || n >= p.n) return;
        char* out = static_cast<char*>(p.out) + ((first + row) * p.ldo + n) * ES;
        if (vec) {
          store4<E>(out, v);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (n + i < p.n) store1<E>(out + i * ES, v[i]);
        }
      };
      if constexpr (WK == 1) {
#pragma unroll
        for (int fm = 0; fm < FM; ++fm)
#pragma unroll
          for (int fn = 0; fn < FN; ++fn) store(acc[fm][fn], fm, fn, wn);
      } else {
        // Join the WK sums of every fragment in wave order: fragment id (fm, fn, wn) is summed by wave id % NW.
        // The barriers leave the copies in flight alone.
        f32x4_t* red = reinterpret_cast<f32x4_t*>(smem + T::RING_BYTES);
#pragma unroll
        for (int fm = 0; fm < FM; ++fm)
#pragma unroll
          for (int fn = 0; fn < FN; ++fn) red[((wk * T::FRAGS) + (fm * FN + fn) * WN + wn) * 64 + lane] = acc[fm][fn];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        compiler_fence();
        for (int id = wave; id < T::FRAGS; id += T::NW) {
          f32x4_t v = red[id * 64 + lane];
#pragma unroll
          for (int x = 1; x < WK; ++x) v += red[(x * T::FRAGS + id) * 64 + lane];
          store(v, id / WN / FN, id / WN % FN, id % WN);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        compiler_fence();
      }
    } else {
      // silu(gate) * up; a row's 128 columns are four waves' two fragments, whose maxima meet in LDS.
      uint32_t* tops = reinterpret_cast<uint32_t*>(smem + T::RING_BYTES);  // [row][8]
#pragma unroll
      for (int fm = 0; fm < FM; ++fm)
#pragma unroll
        for (int fn = 0; fn < FN / 2; ++fn) {
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            acc[fm][fn][i] = gated(acc[fm][fn][i], acc[fm][fn + FN / 2][i]);
            top = max(top, abs_bits(acc[fm][fn][i]));
          }
          top = max(top, (uint32_t)__shfl_xor((int)top, 16));
          top = max(top, (uint32_t)__shfl_xor((int)top, 32));
          if (lane < 16) tops[(fm * 16 + lane) * 8 + wn * (FN / 2) + fn] = top;
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      compiler_fence();
#pragma unroll
      for (int fm = 0; fm < FM; ++fm) {
        const int row = fm * 16 + frag_row;
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, tops[row * 8 + i]);
        const float amax = floored(top), inverse = kE4m3Max / amax;
        if (row >= valid_m) continue;
        if (wn == 0 && lane < 16)
          p.out_scale[(first + row) * p.osm + (int64_t)at.tn * p.osk] = amax / kE4m3Max;
#pragma unroll
        for (int fn = 0; fn < FN / 2; ++fn) {
          const int n = at.tn * T::OUT_COLS + wn * 8 * FN + fn * 16 + group * 4;
          if (n < f)
            *MOEGEMM_GLOBAL(int32_t, static_cast<uint8_t*>(p.out) + (first + row) * p.ldo + n) =
                pack_e4m3(acc[fm][fn] * inverse);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      compiler_fence();
    }
#pragma unroll
    for (int fm = 0; fm < FM; ++fm)
#pragma unroll
      for (int fn = 0; fn < FN; ++fn) acc[fm][fn] = f32x4_t{};
    advance(at);
  }
}

}  // namespace moegemm
