// Which kernel a call's bf16 linears run, and the height of the tiled GEMMs'
// tiles: host rules on sizes alone, free of HIP so that they can be checked
// without a GPU.
#pragma once
#include <stdint.h>

namespace w4a16 {

// A shared-MLP linear (M rows, N output columns, K deep) as the tiled GEMM
// instead of the stream (k_linear_bf16, its weights once per 64 rows).  A
// launch of few tiles takes a tile's time, about 20 us at K = 2816, whatever
// its size; the stream's grows with the 64-row passes and the weights of each.

// The stream on rows in fragment order.  Two passes were never slower; from
// the third on the line is passes times weights.  The FFN block (H = 2816),
// streamed / tiled, in us, at 128, 129, 193..208, 257..288 rows: Im = 512
// 158/173, 164/175, 194/202, 265/259; 1056 163/181, 169/182, 207/209, 240/236;
// 1600 167/183, 201/207, 218/212, 253/238; 2112 176/189, 214/214, 229/217,
// 273/244; 4096 199/208, 225/210, 276/235, 331/266; 12288 300/299, 360/322.
inline bool linear_tiled_frag(int64_t M, int64_t N, int64_t K) {
  return M > 128 && ((M + 63) / 64 - 2) * (N * K) > 4600000;
}

// The stream on row-major rows (16 x 64 bytes a load): tiled earlier.  Im =
// 1056 at 96 / 128 / 160 rows 170/182, 218/219, 228/223; 1600 at 81 / 96
// 178/179, 185/183; 2112 at 65 / 81 / 300 181/187, 187/186, 331/246; 4096 at
// 65 211/204.
inline bool linear_tiled_rows(int64_t M, int64_t N, int64_t K) {
  return (M > 64 && M * N * K > 420000000) || linear_tiled_frag(M, N, K);
}

// The block's two linears (H x Im) stream fragment-order rows: from 17 rows
// on, one row tile gains nothing; `fits`: the padded rows fit in the place
// they are held.
inline bool ffn_fragment_rows(int64_t M, int64_t H, int64_t Im, bool fits, bool tiles_supported) {
  return M > 16 && fits && !(tiles_supported && linear_tiled_frag(M, Im, H));
}

// The tile height, in 32-row blocks, of a launch whose tiles (256 weight rows
// each) are all alike and run one per CU: the time is the rounds of tiles times
// a tile's, cost[blocks - 1].
inline int cheapest_blocks(int64_t M, int64_t wrows, int cus, int max_blocks, const int* cost) {
  const int64_t n_nt = (wrows + 255) / 256;
  int best = 0;
  int64_t least = 0;
  for (int mb = 1; mb <= max_blocks; ++mb) {
    const int64_t tiles = (M + 32 * mb - 1) / (32 * mb) * n_nt;
    const int64_t c = (tiles + cus - 1) / cus * cost[mb - 1];
    if (best == 0 || c < least) {
      best = mb;
      least = c;
    }
  }
  return best;
}

// Dense bf16 GEMM: a tile's time is close to (blocks + 1), its MFMAs and a
// stage's weights, barrier and waits whatever the height.  The FFN block (Im =
// 2112, flat routing) with 1 .. 5 blocks: 287 / 265 / 270 / 283 / 288 us at 512
// rows (2 picked), 399 / 354 / 336 / 346 / 353 at 1024 (3), 572 / 521 / 480 /
// 490 / 468 at 2048 (gate/up 5, down 3: 464).
constexpr int kGemmMaxBlocks = 5;
inline int gemm_bf16_blocks(int64_t M, int64_t wrows, int cus) {
  constexpr int cost[kGemmMaxBlocks] = {2, 3, 4, 5, 6};
  return cheapest_blocks(M, wrows, cus, kGemmMaxBlocks, cost);
}

// The decode streamer's shape for K: k tiles (128 wide) per wavefront in a row
// and wavefronts per sum.  It is also what a sum is: wavefront w's fp32 chain
// over the tiles w tpw .. w tpw + tpw - 1, and those a multiple of ksplit tpw
// behind them, the wavefronts' chains added in order.
struct DecodeShape {
  int tpw;
  int ksplit;
};
inline DecodeShape decode_shape(int64_t K) {
  const int64_t ntiles = (K + 127) / 128;
  if (ntiles <= 2) return {2, 1};
  if (ntiles <= 4) return {4, 1};
  if (ntiles <= 6) return {6, 1};   // down, K = 704: 6 tiles, 4 column groups
  if (ntiles <= 8) return {2, 4};
  if (ntiles <= 16) return {4, 4};
  return {6, 4};                    // gate_up, K = 2816: 22 tiles over 4 wavefronts
}
// whether a chain's tiles lie apart (more than ksplit tpw tiles)
inline bool decode_ranges_interleave(int64_t K) {
  const DecodeShape s = decode_shape(K);
  return (K + 127) / 128 > s.tpw * s.ksplit;
}

// Linear4Bit tiles of at most max_blocks: one round of tiles of 1 .. 6 blocks
// measured 31, 37, 44, 52, 61, 72 us at K = 2816, 11.0 .. 25.4 at K = 704 (a
// stage's barrier and waits dominate few blocks).
constexpr int kLinearW4MaxBlocks = 6;
inline int linear_w4_blocks(int64_t M, int64_t N, int cus, int max_blocks) {
  constexpr int cost[kLinearW4MaxBlocks] = {31, 37, 44, 52, 61, 72};
  return cheapest_blocks(M, N, cus, max_blocks, cost);
}

// Dense GEMMs (gemm_dense.hpp): the tiles that are built, 32 mi rows x 32 ni
// operand columns by kg groups of wavefronts, with the workgroups that share a
// CU and what a stage of 32 k takes, in ns, for a group alone on a CU and for
// each of several (256 .. 1024 tiles of K = 64, 512 and 2816): dy W, dy^T x and
// x W^T.  Only tiles that the rule takes are here.
#define W4A16_DG_TILES_NN(X) \
  X(8, 8, 1, 1, 750, 775)    \
  X(8, 6, 1, 1, 590, 595)    \
  X(6, 8, 1, 1, 570, 575)    \
  X(6, 6, 1, 2, 460, 435)    \
  X(8, 4, 1, 2, 410, 413)    \
  X(4, 8, 1, 2, 450, 408)    \
  X(6, 4, 1, 2, 350, 325)    \
  X(4, 6, 1, 2, 370, 319)    \
  X(4, 4, 1, 2, 290, 243)    \
  X(4, 4, 2, 1, 290, 255)    \
  X(4, 2, 1, 3, 210, 190)    \
  X(2, 4, 1, 3, 205, 178)    \
  X(2, 4, 2, 1, 205, 167)    \
  X(2, 2, 1, 4, 160, 130)    \
  X(2, 2, 4, 1, 160, 118)
#define W4A16_DG_TILES_TN(X) \
  X(8, 8, 1, 1, 730, 730)    \
  X(8, 6, 1, 1, 550, 570)    \
  X(6, 6, 1, 2, 425, 412)    \
  X(8, 4, 1, 2, 400, 380)    \
  X(6, 4, 1, 2, 320, 294)    \
  X(4, 4, 1, 2, 250, 215)    \
  X(4, 4, 2, 1, 250, 210)    \
  X(4, 2, 1, 3, 170, 150)    \
  X(2, 4, 1, 3, 175, 155)    \
  X(2, 4, 2, 1, 175, 138)    \
  X(2, 2, 1, 4, 138, 100)    \
  X(2, 2, 4, 1, 138, 93)
#define W4A16_DG_TILES_NT(X) \
  X(8, 8, 1, 1, 670, 670)    \
  X(8, 6, 1, 1, 520, 520)    \
  X(6, 8, 1, 1, 525, 525)    \
  X(6, 6, 1, 1, 460, 460)    \
  X(8, 4, 1, 1, 420, 420)    \
  X(6, 4, 1, 1, 320, 320)    \
  X(4, 4, 1, 1, 235, 235)    \
  X(4, 2, 1, 2, 145, 135)    \
  X(2, 4, 1, 2, 160, 140)    \
  X(2, 2, 1, 3, 97, 90)

// Products of few rows run as the weights' stream (gemm_thin.hpp), 32 rows x
// `cols` columns a workgroup: up to 64 rows, and up to 512 while the workgroups
// are one round of the CUs (tiles of any shape, split as is best for them / streamed,
// 2816 -> 2816: x W^T 96 rows 12.2/11.7 us; dy W 32 rows 11.5/9.9, 64 12.1/9.3,
// 128 14.2/15.2; 2816 -> 2112, 96 rows 10.9/7.2, 12.3/8.5, 128 11.6/11.6,
// 12.8/13.0; two pairs of 2112, 64 rows 14.3/12.2; 2816 -> 512, 512 rows
// 10.8/7.1, 11.9/8.2; but 512 -> 128, 2048 rows 5.0/6.8, 5.7/7.2: every 32 rows
// read the weights).
inline bool dense_thin(int64_t rows, int64_t n, int cols, int cus) {
  return rows <= 64 || (rows <= 512 && (rows + 31) / 32 * ((n + cols - 1) / cols) <= cus);
}
struct DenseShape {
  int64_t rows, cols;  // of the product (gate/up: both halves' columns)
};
struct DensePlan {
  int mi, ni, kg, ksplit;
};
// planes of fp32 partial sums that a split product may take: at most 8, at
// most 32 MB
constexpr int kDgMaxSplit = 8;
constexpr int64_t kDgPartFloats = int64_t(8) << 20;
inline int dense_part_planes(int64_t plane) {
  const int64_t n = plane > 0 ? kDgPartFloats / plane : 0;
  return n >= kDgMaxSplit ? kDgMaxSplit : n >= 2 ? (int)n : 1;
}
// The tile and split whose time comes out least: rounds of the workgroups that
// fit at once, each nk stages and an epilogue of some 110 ns per 16 x 16 tiles
// of a wavefront (130 where a workgroup has its CU alone); a split's launch that
// adds its planes takes 3 us and their bytes at 4 TB/s.  At the model's shapes
// (100 .. 8192 rows) the plan's tile is within 6 % of the fastest measured.
enum { kPlanNT = 0, kPlanNN = 1, kPlanTN = 2 };  // launch.hpp's DenseLayout
inline DensePlan dense_plan(const DenseShape* sh, int nprob, int nk, int max_split, int cus, int layout) {
  DensePlan best{0, 0, 1, 1};
  int64_t least = 0, plane = 0;
  for (int i = 0; i < nprob; ++i) plane += sh[i].rows * sh[i].cols;
  auto consider = [&](int mi, int ni, int kg, int occ, int64_t alone, int64_t each) {
    int64_t tiles = 0;
    for (int i = 0; i < nprob; ++i)
      tiles += (sh[i].rows + 32 * mi - 1) / (32 * mi) * ((sh[i].cols + 32 * ni - 1) / (32 * ni));
    for (int ks = 1; ks <= max_split && (ks == 1 || nk >= 2 * ks * kg); ++ks) {
      const int64_t n = (tiles * ks + cus - 1) / cus;  // workgroups a CU gets
      const int64_t stages = (nk + ks * kg - 1) / (ks * kg);
      auto round = [&](int64_t w) {
        const int64_t step = w * kg * each > alone ? w * kg * each : alone;
        return (stages + 2) * step + w * ((ks > 1 ? 300 : occ == 1 ? 130 : 110) + 50 * (kg - 1)) * mi * ni;
      };
      int64_t c = n / occ * round(occ);
      if (n % occ != 0) c += round(n % occ);
      if (ks > 1) c += 3000 + (2 * ks + 1) * plane / 1000;
      if (best.mi == 0 || c < least) {
        best = DensePlan{mi, ni, kg, ks};
        least = c;
      }
    }
  };
#define W4A16_DG(MI_, NI_, KG_, OCC_, ALONE_, EACH_) consider(MI_, NI_, KG_, OCC_, ALONE_, EACH_);
  switch (layout) {
    case kPlanNT: W4A16_DG_TILES_NT(W4A16_DG) break;
    case kPlanTN: W4A16_DG_TILES_TN(W4A16_DG) break;
    default: W4A16_DG_TILES_NN(W4A16_DG) break;
  }
#undef W4A16_DG
  return best;
}

}  // namespace w4a16
