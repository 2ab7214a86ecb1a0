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
// the eight rows of a column, rounded: the second operand of accumulate (the matrix
// units take 16 bits; the sums of weights are of the unrounded ones)
template <typename T>
__device__ __forceinline__ u32x4_t at_pack8(f32x4_t a, f32x4_t b) {
  return u32x4_t{at_pack2<T>(a[0], a[1]), at_pack2<T>(a[2], a[3]), at_pack2<T>(b[0], b[1]), at_pack2<T>(b[2], b[3])};
}

// The weights of a softmax as operands, by their exponents over a running maximum that moves
// where one exceeds kOver, and then makes kTop of the largest.  bf16 has fp32's range.  fp16's
// normal numbers are 2^-14 .. 2^15, the least steps 2^-24: the largest weight lies 2^11 high and
// may grow to 2^15, so that one is off by 2^-36 of it at most, n keys' by n 2^-36 (2^24 keys:
// half a rounding).  With 0 and 8, as in bf16, weights of 2^-25 were lost: a quarter of 2^16
// such keys' in decoding, where one wavefront of four had the key above them.
template <typename T>
struct AtWeight {
  static constexpr float kTop = std::is_same_v<T, __bf16> ? 0.f : 11.f, kOver = std::is_same_v<T, __bf16> ? 8.f : 15.f;
};

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

// over L lanes side by side, each gets the sum
template <int L>
__device__ __forceinline__ float at_sum_over(float v) {
  auto add = [](float x, int y) { return x + __int_as_float(y); };
  auto bits = [](float x) { return __float_as_int(x); };
  v = add(v, __builtin_amdgcn_update_dpp(0, bits(v), 0xB1, 0xF, 0xF, false));   // quad [1,0,3,2]
  v = add(v, __builtin_amdgcn_update_dpp(0, bits(v), 0x4E, 0xF, 0xF, false));   // quad [2,3,0,1]
  v = add(v, __builtin_amdgcn_update_dpp(0, bits(v), 0x141, 0xF, 0xF, false));  // row_half_mirror
  if constexpr (L >= 16) v = add(v, __builtin_amdgcn_update_dpp(0, bits(v), 0x140, 0xF, 0xF, false));  // row_mirror
  if constexpr (L >= 32) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  if constexpr (L >= 64) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  return v;
}

// Two tiles side by side of a product's sums (lane: columns 4 c .. of row r), rounded,
// as lane c's eight columns from at_pair_column(c) on: stores of 16 bytes, 64 of a row
// together, take half the time of 8 as they lie.
template <typename T>
__device__ __forceinline__ u32x4_t at_pair(f32x4_t a, f32x4_t b) {
  const auto lo = __builtin_amdgcn_permlane16_swap(at_pack2<T>(a[0], a[1]), at_pack2<T>(b[0], b[1]), false, false);
  const auto hi = __builtin_amdgcn_permlane16_swap(at_pack2<T>(a[2], a[3]), at_pack2<T>(b[2], b[3]), false, false);
  return u32x4_t{lo[0], hi[0], lo[1], hi[1]};
}
__device__ __forceinline__ int at_pair_column(int c) { return 16 * (c & 1) + 8 * (c >> 1); }

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
__host__ __device__ constexpr int at_swz(int row) {
  return (((row >> 2) ^ (row >> 4)) & 1) | (D >= 128 ? ((row & 3) << 1) | (row & 8) : (row & 2) | ((row >> 1) & 4));
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

// A lane's addresses in a tile: of the scores' tile 0 and of accumulate's first
// four rows.  Four rows on the swizzle has its lowest bit turned.  It touches bits
// that a tile's own address (a multiple of 1024) leaves zero, so a read's address
// is an XOR of the step's base, and no register is kept for it over the steps.
template <int D>
struct AtLane {
  uint32_t row, col;
  __device__ __forceinline__ void init() {
    const int l = threadIdx.x & 63, c = l >> 4, r = l & 15;
    const int k = 8 * (r >> 2) + (r & 3), v = 8 * c + (r >> 2);
    row = k * D * 2 + 16 * (at_chunk(0, c) ^ at_swz<D>(k));
    col = v * D * 2 + 16 * (((r & 3) >> 1) ^ at_swz<D>(v)) + 8 * (r & 1);
  }
  // half (0, 1) of D: scores' sum
  __device__ __forceinline__ void half_rows(int half) {
    static_assert(D >= 256, "whole windows");
    row += half * D;
  }
  // half of D: accumulate's columns
  __device__ __forceinline__ void half_cols(int half) {
    if constexpr (D >= 256)
      col += half * D;
    else
      col ^= half * D;
  }
};
// the addresses in the tile at `base`
template <int D>
struct AtRows {
  uint32_t p[2];
  __device__ __forceinline__ AtRows(const AtLane<D>& ln, uint32_t base) {
    p[0] = base + ln.row;
    p[1] = (p[0] ^ 16) + 8 * D;
  }
  __device__ __forceinline__ u32x4_t get(int t, int i) const {
    return *(const lds_u32x4_t*)((p[t] ^ (64 * (i & 3))) + 256 * (i >> 2));
  }
};
template <int D>
struct AtCols {
  uint32_t p[2];
  __device__ __forceinline__ AtCols(const AtLane<D>& ln, uint32_t base) {
    p[0] = base + ln.col;
    p[1] = (p[0] ^ 16) + 8 * D;
  }
  __device__ __forceinline__ u32x4_t get(int d) const {
    const u32x2_t lo = at_tr_read((lds_at4_t*)((p[0] ^ (32 * (d & 7))) + 256 * (d >> 3)));
    const u32x2_t hi = at_tr_read((lds_at4_t*)((p[1] ^ (32 * (d & 7))) + 256 * (d >> 3)));
    return u32x4_t{lo.x, lo.y, hi.x, hi.y};
  }
};

// The products' fragments are read AHEAD of their instructions (the scheduling
// barriers keep them so: a fragment's N instructions take 16 N cycles, its read
// about 130), over the border between the two: `next` is the scores' first.
// Steps of one address come one after the other: it is not kept for later.
template <int NI>
__device__ __forceinline__ constexpr int at_row_step(int j) {
  constexpr int n = NI < 4 ? 1 : NI / 4;
  return NI < 4 ? j >> 1 : 4 * ((j >> 1) % n) + (j >> 1) / n;
}
template <int ND>
__device__ __forceinline__ constexpr int at_col_step(int j) {
  constexpr int n = ND < 8 ? 1 : ND / 8;
  return ND < 8 ? j : 8 * (j % n) + j / n;
}
// s[t][n] = rows of the tile . columns b[n], over 32 NI columns of D from the one
// that the lane's addresses stand at
template <int NI, int AHEAD, int D>
__device__ __forceinline__ void at_scores_first(const AtLane<D>& ln, uint32_t tile, u32x4_t (&next)[AHEAD]) {
  const AtRows<D> rows(ln, tile);
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) next[j] = rows.get(j & 1, at_row_step<NI>(j));
}
template <typename T, int AHEAD, int D, int NI, int N>
__device__ __forceinline__ void at_scores(const AtLane<D>& ln, uint32_t tile, const u32x4_t (&b)[N][NI],
                                          f32x4_t (&s)[2][N], u32x4_t (&a)[AHEAD]) {
  const AtRows<D> rows(ln, tile);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int n = 0; n < N; ++n) s[t][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < 2 * NI; ++j) {
#pragma unroll
    for (int n = 0; n < N; ++n) s[j & 1][n] = at_mfma<T>(a[j % AHEAD], b[n][at_row_step<NI>(j)], s[j & 1][n]);
    if (j + AHEAD < 2 * NI) a[j % AHEAD] = rows.get((j + AHEAD) & 1, at_row_step<NI>(j + AHEAD));
    __builtin_amdgcn_sched_barrier(0);
  }
}
// acc[d][n] += (tile's columns 16 d ..)^T . p[n], ND of D / 16; then the first
// fragments of the tile `of`
template <typename T, int NI, int AHEAD, int D, int ND, int N>
__device__ __forceinline__ void at_accumulate(const AtLane<D>& ln, uint32_t tile, const u32x4_t (&p)[N],
                                              f32x4_t (&acc)[ND][N], uint32_t of, u32x4_t (&next)[AHEAD]) {
  static_assert(ND >= AHEAD, "fragments ahead");
  const AtCols<D> cols(ln, tile);
  const AtRows<D> rows(ln, of);
  u32x4_t a[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) a[j] = cols.get(at_col_step<ND>(j));
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < ND; ++j) {
    const int d = at_col_step<ND>(j);
#pragma unroll
    for (int n = 0; n < N; ++n) acc[d][n] = at_mfma<T>(a[j % AHEAD], p[n], acc[d][n]);
    const int k = j + AHEAD - ND;
    if (k < 0)
      a[j % AHEAD] = cols.get(at_col_step<ND>(j + AHEAD));
    else
      next[k] = rows.get(k & 1, at_row_step<NI>(k));
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Tiles of 32 rows of a matrix of D columns, into LDS by direct loads of NW
// wavefronts.  A cursor goes over the rows in scalar registers: an address from the
// row's number took 300 cycles of a step.
template <int D, int NW>
struct AtFeed {
  static constexpr int kLoads = D / 16 / NW;  // 1 KB loads of a tile, per wavefront
  static_assert(kLoads * NW * 16 == D, "every wavefront as many");
  static constexpr int kStep = 512 / D * NW;  // rows between a wavefront's loads
  int wave, one;                              // one: bytes from row to row
  const unsigned char *matrix, *p;            // p: the next tile's first row
  int left;                                   // rows from there on
  int off, ch;  // a lane's of the first load: bytes to its row, in the row

  __device__ __forceinline__ void init(const unsigned char* m, int64_t stride_bytes, int wave_) {
    wave = wave_;
    one = __builtin_amdgcn_readfirstlane((int)stride_bytes);
    matrix = p = m;
    left = 0;
    const int lane = threadIdx.x & 63, row = 512 / D * wave + lane / (D / 8);
    off = row * one;
    ch = 16 * ((lane % (D / 8)) ^ at_swz<D>(row));
  }
  // to row `first` of `rows`, `more` bytes further
  __device__ __forceinline__ void seek(int first, int rows, int64_t more = 0) {
    p = matrix + (int64_t)first * one + more;
    left = rows - first;
  }
  // tiles on (n may be negative)
  __device__ __forceinline__ void skip(int n) {
    p += (int64_t)(32 * n) * one;
    left -= 32 * n;
  }
  // The next tile's rows (past the last, it again; none, or !any: nothing is read).
  __device__ __forceinline__ void issue(unsigned char* tile, bool any) const {
    const int last = any ? left - 1 : -1;
    const auto rsrc = make_rsrc(p, last < 0 ? 0u : 0x7FFFFFFFu);
    tile += 1024 * wave;
    // rows past the first load's are other bits of the row: so is their swizzle
    // (opaque: no register is kept for each load over the steps)
    const int c0 = (int)opaque((uint32_t)ch);
    if (last >= 31) {
#pragma unroll
      for (int j = 0; j < kLoads; ++j)
        px_dma16(rsrc, off + (c0 ^ (16 * at_swz<D>(kStep * j))), kStep * j * one, tile + 1024 * NW * j);
    } else {
      const int row = 512 / D * wave + (int)opaque(threadIdx.x & 63) / (D / 8);
#pragma unroll
      for (int j = 0; j < kLoads; ++j)
        px_dma16(rsrc, min(row + kStep * j, last) * one + (c0 ^ (16 * at_swz<D>(kStep * j))), 0, tile + 1024 * NW * j);
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

// Registers that loads in flight will fill, waited for here: in a loop the compiler
// would wait in every step, and with them for the steps' loads issued since.
template <int M, int N>
__device__ __forceinline__ void at_settle(u32x4_t (&x)[M][N]) {
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int n = 0; n < N; ++n) asm volatile("" : "+v"(x[m][n]));
}
template <int N>
__device__ __forceinline__ void at_settle(float (&x)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) asm volatile("" : "+v"(x[n]));
}

// The keys lo .. hi - 1 that the queries first .. last of a sequence see, one at least
__device__ __forceinline__ void at_seen_keys(const AttnArgs& a, int nk, int off, int first, int last, int& lo,
                                             int& hi) {
  hi = a.causal ? min(nk, last + off + 1) : nk;
  lo = a.window > 0 ? max(0, first + off - a.window + 1) : 0;
}

// Whether query `q` sees a key at all.  One that does and has a sum of zero saw scores of
// -infinity alone: its softmax is not a number.
__device__ __forceinline__ bool at_sees(const AttnArgs& a, int nk, int off, int q) {
  return nk > 0 && (!a.causal || q + off >= 0);
}

// The tile of `rows` rows that workgroup item `rank` has.  Tiles go by level,
// the tiles of their sequence in front of them, the highest first: with a causal
// mask a tile's work grows with it, and what runs last should be short (more
// sequences than lanes: one sequence after the other).  Behind the sequences the
// rows past the last are one more (seq = n).  first, len: the sequence's rows;
// offsets are held to 0 .. total, whatever the array says.  The search takes 2000
// cycles, which a sequence alone need not wait for (heads of 512, both timed in turn:
// gradients of 1024 tokens 179.5 -> 173.0 us, of 4096 1411 -> 1400; forward 253.5 -> 251).
struct AtItem {
  int seq, level, tiles, first, len;
};
__device__ __forceinline__ int at_wave_sum(int v) {
  return (int)dpp_wave_reduce((uint32_t)v, [](uint32_t x, uint32_t y) { return x + y; });
}
__device__ __forceinline__ AtItem at_find(const int32_t* __restrict__ cu, int n, int total, int rows, int rank) {
  const int lane = threadIdx.x & 63;
  AtItem it{-1, 0, 0, 0, 0};
  for (int base = 0; base <= n; base += 64) {
    const int b = base + lane;
    int first = total, end = total;
    if (b <= n) first = min(max(cu[b], 0), total);
    if (b < n) end = min(max(cu[b + 1], first), total);
    const int len = end - first, tiles = (len + rows - 1) / rows;
    const int all = at_wave_sum(tiles);
    if (rank >= all) {
      rank -= all;
      continue;
    }
    int at;
    if (n == 1) {
      const int own = __builtin_amdgcn_readlane(tiles, 0);
      at = rank < own ? 0 : 1;
      it.level = at == 0 ? own - 1 - rank : rank - own;
    } else if (n < 64) {
      // the highest level at or above which there are more than `rank` tiles
      int low = 0, high = (int)wave_max_u32((uint32_t)tiles);
      while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (at_wave_sum(max(tiles - mid, 0)) > rank)
          low = mid;
        else
          high = mid;
      }
      it.level = low;
      const int k = rank - at_wave_sum(max(tiles - low - 1, 0));
      const unsigned long long has = __ballot(tiles > low);
      const bool mine = tiles > low && __popcll(has & ((1ull << lane) - 1ull)) == k;
      at = __ffsll((unsigned long long)__ballot(mine)) - 1;
    } else {
      int sum = tiles;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(sum, o);
        if (lane >= o) sum += v;
      }
      at = __ffsll((unsigned long long)__ballot(sum > rank)) - 1;
      it.level = __builtin_amdgcn_readlane(sum, at) - 1 - rank;
    }
    it.seq = base + at;
    it.tiles = __builtin_amdgcn_readlane(tiles, at);
    it.first = __builtin_amdgcn_readlane(first, at);
    it.len = __builtin_amdgcn_readlane(len, at);
    return it;
  }
  return it;
}
// a sequence's rows, as at_find holds them
__device__ __forceinline__ void at_rows(const int32_t* __restrict__ cu, int n, int total, int seq, int& first,
                                        int& len) {
  first = total;
  len = 0;
  if (seq < n) {
    first = min(max(cu[seq], 0), total);
    len = min(max(cu[seq + 1], first), total) - first;
  }
}

// The rows of a workgroup's tile (low: where there are few of them), and of the other
// axis' steps.
constexpr int attn_rows(int kernel, int D, bool low = false) {
  if (kernel == kAttnForward) return (D == 512 ? 128 : 256) >> (low ? 1 : 0);
  return D == 512 || (low && D > 64) ? 64 : D == 128 ? 192 : 128;
}
constexpr int attn_keys(int kernel, int D) { return kernel == kAttnForward && D < 256 ? 64 : 32; }
constexpr int64_t kAttnParts = 512, kAttnChunk = 12, kAttnMostParts = 32;
// Forward: smaller tiles up to so many of the others and their heads (of 512 as many as
// are ever split: the others' kernel has no registers left for that).
constexpr int64_t attn_low(int64_t D) { return D == 512 ? kAttnParts : kAttnParts / 2; }

// How many workgroups share a tile of `steps` steps over the other axis, and what
// one of them has.  The first parts of all tiles go first: what has no part is last.
// (Quotients come from the vector unit: what loops go by is brought back to scalars.)
__device__ __forceinline__ int at_parts(const AttnArgs& a, int steps) {
  return __builtin_amdgcn_readfirstlane(max(min((steps + a.chunk - 1) / a.chunk, a.split), 1));
}
struct AtPart {
  int index, of, first, steps;
};
__device__ __forceinline__ AtPart at_part(const AttnArgs& a, int steps, int index) {
  AtPart p{index, at_parts(a, steps), 0, 0};
  // its share, and the first steps % of parts one more
  const int each = __builtin_amdgcn_readfirstlane(steps / p.of), more = steps - each * p.of;
  p.first = index * each + min(index, more);
  p.steps = each + (index < more ? 1 : 0);
  return p;
}

// The steps of `keys` keys that a tile of `rows` queries from wg0 on takes: all keys
// that some query of it sees.
struct AtSpan {
  int lo, hi, steps;
};
__device__ __forceinline__ AtSpan at_key_span(const AttnArgs& a, int nk, int off, int wg0, int rows, int nq, int keys) {
  AtSpan s;
  at_seen_keys(a, nk, off, wg0, min(wg0 + rows, nq) - 1, s.lo, s.hi);
  s.lo &= -keys;
  s.steps = s.hi > s.lo ? (s.hi - s.lo + keys - 1) / keys : 0;
  return s;
}

// A workgroup's head and rank.  Workgroups go round robin to the eight XCDs: each
// has heads of its own where they divide among them, so that the queries' heads
// that share keys and values share an L2.
struct AtPlace {
  int head, rank;
};
__device__ __forceinline__ AtPlace at_place(int heads) {
  const int b = (int)blockIdx.x;
  if ((heads & 7) == 0) {
    const int per = heads >> 3, i = b >> 3;
    return {(b & 7) * per + i % per, i / per};
  }
  return {b % heads, b / heads};
}

}  // namespace w4a16
