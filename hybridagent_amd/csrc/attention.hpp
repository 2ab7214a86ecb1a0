// What the attention kernels share (kernels_attention.hip: packed prompts,
// kernels_attention_back.hip: their gradients, kernels_attention_decode.hip).
//
// All three matrix kernels are one pair of steps on v_mfma_f32_16x16x32 with
// fp32 accumulation, on tiles of 32 rows of [rows][D] in LDS:
//
//   scores      C[32 rows][16 columns] = tile . B^T, B 16 rows of D in registers
//   accumulate  A^T[D][16 columns] += tile^T . C, C as scores left it
//
// Lane l of a wavefront has column l % 16 of C, and of its 32 rows the eight
// 8 c .. 8 c + 7, c = l / 16: row r of the first operand's tile t (t = 0, 1) is
// row 8 (r / 4) + 4 t + r % 4 of the 32.  Rounded and packed these eight are the
// second operand of accumulate as they are: the weights never leave their lane,
// and a column's maximum, sum and factor are one register of its four lanes.
//
//   prompts     tile = keys, values;  columns = queries;  A = out
//   dq          tile = keys, values;  columns = queries;  A = dq
//   dk, dv      tile = queries, dout; columns = keys;     A = dk, dv
#pragma once
#include "common.hpp"
#include "launch.hpp"
#include "lds_pipe.hpp"

namespace w4a16 {

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
typedef __attribute__((ext_vector_type(4))) __bf16 at_bf16x4_t;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// T: a 16-bit type
template <typename T>
__device__ __forceinline__ f32x4_t at_mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (std::is_same_v<T, __bf16>)
    return mfma16(a, b, c);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
}
template <typename T>
__device__ __forceinline__ uint32_t at_pack2(float lo, float hi) {
  if constexpr (std::is_same_v<T, __bf16>) {
    return pack_bf16x2(lo, hi);
  } else {
    const f16x2_t v = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, v);
  }
}
template <typename T>
__device__ __forceinline__ float at_lo(uint32_t w) {
  if constexpr (std::is_same_v<T, __bf16>)
    return bf16_bits_to_f32(w & 0xFFFFu);
  else
    return (float)__builtin_bit_cast(f16x2_t, w).x;
}
template <typename T>
__device__ __forceinline__ float at_hi(uint32_t w) {
  if constexpr (std::is_same_v<T, __bf16>)
    return __uint_as_float(w & 0xFFFF0000u);
  else
    return (float)__builtin_bit_cast(f16x2_t, w).y;
}
// the eight rows of a column, rounded: the second operand of accumulate
template <typename T>
__device__ __forceinline__ u32x4_t at_pack8(f32x4_t a, f32x4_t b) {
  return u32x4_t{at_pack2<T>(a[0], a[1]), at_pack2<T>(a[2], a[3]), at_pack2<T>(b[0], b[1]), at_pack2<T>(b[2], b[3])};
}

// over the four lanes of a column (c = 0 .. 3), each gets the result
template <typename Op>
__device__ __forceinline__ float at_over_c(float v, Op op) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(p[0]), __uint_as_float(p[1]));
  const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float at_max_over_c(float v) {
  return at_over_c(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float at_sum_over_c(float v) {
  return at_over_c(v, [](float x, float y) { return x + y; });
}

// The 16-byte chunk of D that lane group c takes in step i of a score's sum
// (32 columns of D a step, in an order of its own: both operands use it)
__device__ __forceinline__ int at_chunk(int i, int c) { return 4 * i + (((c & 1) << 1) | (c >> 1)); }

// LDS tile [32 rows][D], 16-byte chunks XOR-swizzled by the row so that both
// reads are free of bank conflicts (64 banks of 4 bytes):
//   scores: ds_read_b128, lane l row 8 (r / 4) + 4 t + r % 4 (r = l % 16), chunk
//   at_chunk(i, l / 16), in groups of lanes 0..3, 12..15, 20..27 and 4..11,
//   16..19, 28..31 of each 32;
//   accumulate: ds_read_b64_tr_b16, 32 lanes at rows 8 c + 0 .. 3 (+ 4) of two
//   neighbouring c, two neighbouring chunks.
// Rows are a multiple of the 256-byte window apart, or (D 64) half of one.
template <int D>
__device__ __forceinline__ int at_swz(int row) {
  const int low = ((row >> 2) ^ (row >> 4)) & 1;
  if constexpr (D >= 128)
    return low | ((row & 3) << 1) | (row & 8);
  else
    return low | (row & 2) | ((row >> 1) & 4);
}
template <int D>
constexpr int at_tile_bytes() { return 32 * D * 2; }

typedef __attribute__((address_space(3))) at_bf16x4_t lds_at4_t;
typedef __attribute__((address_space(3))) u32x4_t lds_u32x4_t;
// (restrict: see dg_tr_read)
__device__ __forceinline__ u32x2_t at_tr_read(lds_at4_t* __restrict__ p) {
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(p));
}
__device__ __forceinline__ uint32_t at_lds(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const unsigned char*)p;
}

// A lane's addresses in a tile.  Its swizzle touches bits that a tile's own
// address (a multiple of 1024) leaves zero, so a read's address is one XOR of
// the step's base, which no register is kept for over the steps.
template <int D>
struct AtLane {
  uint32_t row[2];  // scores' tiles
  uint32_t col[2];  // accumulate's halves
  __device__ __forceinline__ void init() {
    const int l = threadIdx.x & 63, c = l >> 4, r = l & 15;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int k = 8 * (r >> 2) + 4 * t + (r & 3);
      row[t] = k * D * 2 + 16 * (at_chunk(0, c) ^ at_swz<D>(k));
      const int v = 8 * c + 4 * t + (r >> 2);
      col[t] = v * D * 2 + 16 * (((r & 3) >> 1) ^ at_swz<D>(v)) + 8 * (r & 1);
    }
  }
  // half (0, 1) of D: scores' sum
  __device__ __forceinline__ void half_rows(int half) {
    static_assert(D >= 256, "whole windows");
    row[0] += half * D;
    row[1] += half * D;
  }
  // half of D: accumulate's columns
  __device__ __forceinline__ void half_cols(int half) {
    if constexpr (D >= 256) {
      col[0] += half * D;
      col[1] += half * D;
    } else {
      col[0] ^= half * D;
      col[1] ^= half * D;
    }
  }
};
// the addresses in the tile at `base`
struct AtRows {
  uint32_t p[2];
  template <int D>
  __device__ __forceinline__ AtRows(const AtLane<D>& ln, uint32_t base) : p{base + ln.row[0], base + ln.row[1]} {}
  __device__ __forceinline__ u32x4_t get(int t, int i) const {
    return *(const lds_u32x4_t*)((p[t] ^ (64 * (i & 3))) + 256 * (i >> 2));
  }
};
struct AtCols {
  uint32_t p[2];
  template <int D>
  __device__ __forceinline__ AtCols(const AtLane<D>& ln, uint32_t base) : p{base + ln.col[0], base + ln.col[1]} {}
  __device__ __forceinline__ u32x4_t get(int d) const {
    const u32x2_t lo = at_tr_read((lds_at4_t*)((p[0] ^ (32 * (d & 7))) + 256 * (d >> 3)));
    const u32x2_t hi = at_tr_read((lds_at4_t*)((p[1] ^ (32 * (d & 7))) + 256 * (d >> 3)));
    return u32x4_t{lo.x, lo.y, hi.x, hi.y};
  }
};

// s[t][n] = rows of the tile . columns b[n], over 32 NI columns of D from the one
// that the lane's addresses stand at.  AHEAD: fragments read ahead of their
// matrix instructions (the scheduling barriers keep them so)
template <typename T, int AHEAD, int D, int NI, int N>
__device__ __forceinline__ void at_scores(const AtLane<D>& ln, uint32_t tile, const u32x4_t (&b)[N][NI],
                                          f32x4_t (&s)[2][N]) {
  const AtRows rows(ln, tile);
  u32x4_t a[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) a[j] = rows.get(j & 1, j >> 1);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int n = 0; n < N; ++n) s[t][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < 2 * NI; ++j) {
#pragma unroll
    for (int n = 0; n < N; ++n) s[j & 1][n] = at_mfma<T>(a[j % AHEAD], b[n][j >> 1], s[j & 1][n]);
    if (j + AHEAD < 2 * NI) a[j % AHEAD] = rows.get((j + AHEAD) & 1, (j + AHEAD) >> 1);
    __builtin_amdgcn_sched_barrier(0);
  }
}
// acc[d][n] += (tile's columns 16 d ..)^T . p[n], as many of D
template <typename T, int AHEAD, int D, int ND, int N>
__device__ __forceinline__ void at_accumulate(const AtLane<D>& ln, uint32_t tile, const u32x4_t (&p)[N],
                                              f32x4_t (&acc)[ND][N]) {
  constexpr int A = ND < AHEAD ? ND : AHEAD;
  const AtCols cols(ln, tile);
  u32x4_t a[A];
#pragma unroll
  for (int d = 0; d < A; ++d) a[d] = cols.get(d);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int d = 0; d < ND; ++d) {
#pragma unroll
    for (int n = 0; n < N; ++n) acc[d][n] = at_mfma<T>(a[d % A], p[n], acc[d][n]);
    if (d + A < ND) a[d % A] = cols.get(d + A);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Two tiles of 32 rows, from matrices of D columns, into an LDS slot by direct
// loads of NW wavefronts.
template <int D, int NW>
struct AtFeed {
  static constexpr int kTileLoads = D / 16;              // 1 KB loads of a tile
  static constexpr int kLoads = 2 * kTileLoads / NW;     // of both, per wavefront
  static constexpr int kSlot = 2 * at_tile_bytes<D>();
  static_assert(kLoads * NW == 2 * kTileLoads, "every wavefront as many");
  static constexpr bool kSplit = kTileLoads < NW;        // a wavefront loads of one tile alone
  static constexpr int kRows = 512 / D;                  // of a load
  static constexpr int kStep = kRows * (kSplit ? kTileLoads : NW);  // rows between a wavefront's loads
  int row, chunk;                                        // a lane's: of the first load
  int64_t stride[2];                                     // bytes
  const unsigned char* p[2];

  __device__ __forceinline__ void init(const unsigned char* p0, int64_t stride0, const unsigned char* p1,
                                       int64_t stride1, int wave) {
    const int lane = threadIdx.x & 63;
    row = kRows * (wave % kTileLoads) + lane / (D / 8);
    chunk = 16 * ((lane % (D / 8)) ^ at_swz<D>(row));
    p[0] = p0;
    p[1] = p1;
    stride[0] = stride0;
    stride[1] = stride1;
  }
  // rows first .. of `rows` in all (past the last, it again; none: nothing is
  // read); more0, more1: bytes in front of the matrices' own first
  __device__ __forceinline__ void issue(unsigned char* slot, int first, int rows, int wave, int64_t more0 = 0,
                                        int64_t more1 = 0) const {
    const int last = rows - 1 - first;
    const bool whole = last >= 31;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      if (kSplit && m != wave / kTileLoads) continue;
      const auto rsrc = make_rsrc(p[m] + first * stride[m] + (m ? more1 : more0), last < 0 ? 0u : 0x7FFFFFFFu);
      unsigned char* to = slot + m * at_tile_bytes<D>() + 1024 * (wave % kTileLoads);
      const int one = (int)stride[m];
#pragma unroll
      for (int j = 0; j < (kSplit ? 1 : kTileLoads / NW); ++j) {
        // rows past the first load's are other bits of the row: so is their swizzle
        const int ch = chunk ^ (16 * at_swz<D>(kStep * j));
        if (whole)
          px_dma16(rsrc, row * one + ch, kStep * j * one, to + 1024 * NW * j);
        else
          px_dma16(rsrc, min(row + kStep * j, last) * one + ch, 0, to + 1024 * NW * j);
      }
    }
  }
};

// 16 rows' worth of second operand: 32 NI columns of row `row` of a matrix
template <int NI>
__device__ __forceinline__ void at_load_row(const void* p, int64_t row, int64_t stride, u32x4_t (&b)[NI]) {
  const unsigned char* q = static_cast<const unsigned char*>(p) + row * stride;
  const int c = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int i = 0; i < NI; ++i) b[i] = ld16(q + 16 * at_chunk(i, c));
}

// The keys lo .. hi - 1 that the queries first .. last of a sequence see, one at least
__device__ __forceinline__ void at_seen_keys(const AttnArgs& a, int nk, int off, int first, int last, int& lo, int& hi) {
  hi = a.causal ? min(nk, last + off + 1) : nk;
  lo = a.window > 0 ? max(0, first + off - a.window + 1) : 0;
}

// The sequence and the tile of `rows` rows in it that workgroup item idx has;
// the tiles of all sequences in their order, then those of the rows behind the
// last sequence (seq = n).  first, len: the sequence's rows.  Offsets are held
// to 0 .. total, whatever the array says.
struct AtItem {
  int seq, tile, tiles, first, len;
};
__device__ __forceinline__ AtItem at_find(const int32_t* __restrict__ cu, int n, int total, int rows, int idx) {
  const int lane = threadIdx.x & 63;
  AtItem it{-1, 0, 0, 0, 0};
  for (int base = 0; base <= n; base += 64) {
    const int b = base + lane;
    int first = total, end = total;
    if (b <= n) first = min(max(cu[b], 0), total);
    if (b < n) end = min(max(cu[b + 1], first), total);
    const int len = end - first, tiles = (len + rows - 1) / rows;
    int sum = tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o);
      if (lane >= o) sum += v;
    }
    const int all = __builtin_amdgcn_readlane(sum, 63);
    if (idx < all) {
      const int at = __ffsll((unsigned long long)__ballot(sum > idx)) - 1;
      it.seq = base + at;
      it.tiles = __builtin_amdgcn_readlane(tiles, at);
      it.tile = idx - (__builtin_amdgcn_readlane(sum, at) - it.tiles);
      it.first = __builtin_amdgcn_readlane(first, at);
      it.len = __builtin_amdgcn_readlane(len, at);
      return it;
    }
    idx -= all;
  }
  return it;
}
// a sequence's rows, as at_find holds them
__device__ __forceinline__ void at_rows(const int32_t* __restrict__ cu, int n, int total, int seq, int& first, int& len) {
  first = total;
  len = 0;
  if (seq < n) {
    first = min(max(cu[seq], 0), total);
    len = min(max(cu[seq + 1], first), total) - first;
  }
}

// workgroup -> item: every XCD (workgroups go round robin) has a run of
// consecutive ones, so that the heads that share keys and values share an L2
__device__ __forceinline__ int at_swizzle(int total) {
  const int per = (total + 7) >> 3;
  const int i = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
  return (int)(blockIdx.x >> 3) < per && i < total ? i : -1;
}
inline unsigned at_grid(int64_t total) { return (unsigned)((total + 7) / 8 * 8); }

}  // namespace w4a16
