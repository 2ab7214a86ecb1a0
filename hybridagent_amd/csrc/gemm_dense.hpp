// Dense bf16 GEMM of the training forms (gated_mlp, HybridLink): one kernel
// template for the three products that a linear y = x W^T takes part in,
//
//   kDgNT  y  = x W^T    both operands with k contiguous
//   kDgNN  dx = dy W     the rows with k contiguous, the weights [k][n]
//   kDgTN  dW = dy^T x   both operands [k][.], k the tokens
//
// as C[m][n] = sum_k A(m, k) B(n, k) with fp32 accumulation on
// v_mfma_f32_16x16x32_bf16, B the first operand, so that a lane ends with
// four consecutive n of one row m.
//
// A workgroup of four wavefronts (2 x 2) owns a tile of 32 MI rows x 32 NI
// columns, a wavefront 16 MI x 16 NI of it; with KG > 1 (dy W and dy^T x) there
// are KG such groups, each with a part of K and a ring of its own, whose sums
// are added in LDS (a few hundred rows: a wavefront's chain of stages is what
// takes the time).  k advances in stages of 32 through a ring of dg_slots LDS
// slots filled by direct 16-byte global -> LDS loads; the fragments of stage
// t + 1 are read while stage t is multiplied, so that a slot has one barrier and
// its loads have two to three stages to land.  Slots past the end are issued
// with an empty buffer descriptor, which reads nothing, so that every wait
// counts the same loads.
//
// A slot is a stage; in x W^T two, so that each row comes in whole 128-byte
// lines: half a line per stage has left the L1 before the other half is asked
// for, and the line comes from the L2 twice (2816 -> 2816, one / two stages a
// slot: 1024 rows 28.4/23.9 us, 2049 38.9/34.5; 8192 rows 2816 -> 4224
// 180.6/162.0).  dy W, one of whose operands has rows, loses by it (2049 rows
// 38.5/42.0: longer stages take more LDS or land later).
//
// Bound: many rows: the matrix units at the clock that the card holds under
// them (2816 -> 4224 of 8192 rows 162 us, 1200 TFLOP/s; dy W 2816 -> 2112 85 us,
// 1150; dy^T x 2112 x 2816 of 8192 rows 101 us, 960); hundreds (2816 -> 2816 of
// 1024 rows 23.9 us, 680): no unit by itself.  With a wavefront or two per SIMD,
// LDS reads, loads and MFMAs overlap in part (of the CUs' cycles in 193 .. 2049 rows
// the matrix units have 0.19 .. 0.47, LDS reads 0.17 .. 0.27, the wavefronts wait
// in 0.14 .. 0.42), and 132 .. 198 workgroups leave CUs idle.  The tile and the
// split are dense_plan's (rules.hpp).
//
// LDS formats of a slot's operand tile, both free of bank conflicts:
//   rows  (k contiguous)  [rows][32 or 64 k], the 16-byte chunks of a row
//         XOR-swizzled by bits of the row (dg_row_swz; 64 k: row / 2): a fragment
//         is 16 rows x 64 bytes, one ds_read_b128 per lane;
//   cols  ([k][.])        [32 k][cols], the 32-byte units of a row
//         XOR-swizzled by bits of k (dg_swz): a fragment of 16 columns x 32 k
//         is two transposing reads (ds_read_b64_tr_b16), which take 4 k x 16
//         columns per 16 lanes and give each lane the 4 k of its column.
// The swizzle is applied to the load's source address (a direct load's LDS
// addresses are consecutive).
#pragma once
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"
#include "lds_pipe.hpp"
#include "rules.hpp"

namespace w4a16 {

constexpr int kDgThreads = 256;
constexpr int kDgKT = 32;     // k per stage

// Whether a slot of the ring is two stages
constexpr bool dg_pairs(int layout) { return layout == kDgNT; }
constexpr int dg_slot_bytes(int layout, int mi, int ni) {
  return 32 * (mi + ni) * kDgKT * 2 * (dg_pairs(layout) ? 2 : 1);
}
// LDS slots of a tile: four, or three where two workgroups then share a CU.
// Pairs of stages: three where they fit in tiles of few MFMAs a stage, else two
// (2049 rows 2816 -> 2816, two / three: 6 x 4 tiles 40.5/36.1 us, 6 x 6 45.9/46.6;
// 6144 rows -> 2048, 6 x 4 tiles 59.6/65.9, two workgroups of which no longer
// share a CU, but 6 x 8 take 53).
constexpr int dg_slots(int layout, int mi, int ni, int kg) {
  if (dg_pairs(layout)) return mi * ni <= 24 && 3 * kg * dg_slot_bytes(layout, mi, ni) <= 160 * 1024 ? 3 : 2;
  return mi * ni >= 24 && mi * ni <= 36 ? 3 : 4;
}
constexpr int kDgGroupM = 4;  // row tiles that run with a column tile
constexpr int dg_bm(int mi) { return 32 * mi; }
constexpr int dg_bn(int epi, int ni) { return epi == kDgGateUp ? 16 * ni : 32 * ni; }

// the epilogue's LDS rows (in the ring's place, behind what the groups left):
// floats between them, 4 modulo the 64 banks where that is not twice the row
constexpr int dg_epi_pitch(int no) { return no > 4 ? 132 : no > 2 ? 68 : 16 * no + 4; }

typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4_t;

// s_waitcnt vmcnt(N), nothing else
template <int N>
__device__ __forceinline__ void dg_wait_vm() {
  __builtin_amdgcn_s_waitcnt(px_vm_wait(N));
}

// A transposing LDS read: of 4 k x 16 columns per 16 lanes (lane i's address:
// row i / 4, columns 4 (i % 4) .. + 3) each lane gets the 4 k of column i.  The
// restrict argument gives the read alias information: without any the compiler
// waits for every direct LDS load in flight before it.
typedef __attribute__((address_space(3))) bf16x4_t lds_bf16x4_t;
__device__ __forceinline__ bf16x4_t dg_tr_read(lds_bf16x4_t* __restrict__ p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16(p);
}

// the swizzle of row k of a cols tile of W columns: which 32-byte unit of an
// aligned group goes where.  A transposing read's first 32 lanes take rows 0 ..
// 3 and 8 .. 11 (+ 4): eight different units of the 256-byte bank window.
template <int W>
__device__ __forceinline__ int dg_swz(int k) {
  if constexpr (W % 128 == 0)
    return (k & 3) | ((k >> 1) & 4);
  else  // rows are 128 bytes apart modulo the window
    return ((k >> 1) & 1) | ((k >> 2) & 2);
}

// the swizzle of the 16-byte chunks of a rows tile, by the row's group of four.
// A 16-byte read goes in groups of 16 lanes, 0..3, 12..15, 20..27 and 4..11,
// 16..19, 28..31 of each 32: with lane l on row l % 16, chunk l / 16, each such
// group covers the 256-byte bank window once.
__device__ __forceinline__ int dg_row_swz(int quad) { return (((quad ^ (quad >> 1)) & 1) << 1) | ((quad >> 1) & 1); }

// One operand's side of a tile: W rows (or columns), F fragments of 16 per
// wavefront.  COLS: the cols format.  GU (rows format): the first half of a
// wavefront's fragments come from p, the second half, same rows, from p2.
// PAIR: rows format of two stages.
template <bool COLS, bool GU, int F, bool PAIR>
struct DgOperand {
  static constexpr int W = 32 * F;
  static constexpr int kBytes = W * kDgKT * (PAIR ? 4 : 2);  // of a stage, or pair of stages
  static constexpr int kLoads = PAIR ? F : F / 2;            // per wavefront, of the same
  int voff[kLoads];                     // a lane's source bytes, per load
  int foff[COLS ? F : PAIR ? 2 : 1];    // its fragment bytes in a stage

  // first: the tile's first row, n: rows there are (rows past it repeat the last)
  __device__ __forceinline__ void init(int first, int n, int64_t ld, int wave) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int ins = wave + 4 * j;
      if constexpr (COLS) {
        const int pos = 1024 * ins + 16 * lane;
        const int k = pos / (2 * W), s = (pos - k * 2 * W) >> 4;
        const int unit = (s >> 1) ^ dg_swz<W>(k);
        const int col = min(16 * unit + 8 * (s & 1), n - first - 8);
        voff[j] = k * (int)ld * 2 + 2 * col;
      } else {
        int r = PAIR ? 8 * ins + (lane >> 3) : 16 * ins + (lane >> 2);
        const int chunk = PAIR ? (lane & 7) ^ ((r >> 1) & 7) : (lane & 3) ^ dg_row_swz((lane >> 4) & 3);
        if constexpr (GU) {
          // tile rows 16 F w + [0, 8 F): rows 8 F w + .. of p, [8 F, 16 F): of p2
          const int w = r / (16 * F), in = r - 16 * F * w;
          r = 8 * F * w + (in >= 8 * F ? in - 8 * F : in);
        }
        voff[j] = min(r, n - first - 1) * (int)ld * 2 + 16 * chunk;
      }
    }
  }
  // w: the wavefront's half of the tile
  __device__ __forceinline__ void init_frag(int w) {
    const int lane = threadIdx.x & 63;
    if constexpr (COLS) {
      const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);
#pragma unroll
      for (int f = 0; f < F; ++f) foff[f] = k * 2 * W + 32 * ((w * F + f) ^ dg_swz<W>(k)) + 8 * (lane & 3);
    } else if constexpr (PAIR) {
      foff[0] = 2048 * F * w + (lane & 15) * 128 + 16 * ((lane >> 4) ^ ((lane >> 1) & 7));
      foff[1] = foff[0] ^ 64;
    } else {
      foff[0] = 1024 * F * w + (lane & 15) * 64 + 16 * ((lane >> 4) ^ dg_row_swz((lane >> 2) & 3));
    }
  }
  static __device__ __forceinline__ bool second(int j, int wave) {
    return (wave + 4 * j) / (PAIR ? 2 : 1) % F >= F / 2;
  }
  // h: the stage of a pair
  __device__ __forceinline__ u32x4_t frag(const unsigned char* st, int f, int h) const {
    if constexpr (COLS) {
      const unsigned char* p = st + foff[f];
      const bf16x4_t lo = dg_tr_read((lds_bf16x4_t*)p);
      const bf16x4_t hi = dg_tr_read((lds_bf16x4_t*)(p + 8 * W));
      const bf16x8_t v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(u32x4_t, v);
    } else if constexpr (PAIR) {
      return *reinterpret_cast<const u32x4_t*>(st + foff[h] + 2048 * f);
    } else {
      return *reinterpret_cast<const u32x4_t*>(st + foff[0] + 1024 * f);
    }
  }
};

// ---- epilogues on eight consecutive columns n .. n + 7 of row m

__device__ __forceinline__ void dg_unpack8(u32x4_t u, float v[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf16_bits_to_f32(w[i] & 0xFFFFu);
    v[2 * i + 1] = bf16_bits_to_f32(w[i] >> 16);
  }
}
__device__ __forceinline__ u32x4_t dg_pack8(const float v[8]) {
  return u32x4_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}

// What an epilogue reads and writes, from a row on: buffers that end with the
// problem's last row, so that elements past it (and kDgOut) read as zero and
// are not written.  Element offsets o of a row-major [rows][N] (at most 256
// rows of 32768: byte offsets below 2^25).
struct DgTarget {
  __amdgpu_buffer_rsrc_t out, out2, sum, sum2, in, bias, part, part2;
  bool keep;  // kDgGateUp: sum, sum2 wanted
};
constexpr int kDgOut = 1 << 28;
__device__ __forceinline__ DgTarget dg_target(const DgArgs& a, const DgProblem& p, int split, int row, int rows,
                                              bool two) {
  const int left = max(min(p.M - row, rows), 0);
  const int64_t at = (int64_t)row * p.N;
  const uint32_t bytes = (uint32_t)(left * p.N) * 2u;
  auto at16 = [&](const uint16_t* q) { return make_rsrc(q + at, q != nullptr ? bytes : 0u); };
  auto at32 = [&](const float* q) { return make_rsrc(q + at, q != nullptr ? 2u * bytes : 0u); };
  DgTarget g;
  g.out = at16(p.e.out);
  g.out2 = at16(p.e.out2);
  g.sum = at32(p.e.sum);
  g.sum2 = at32(p.e.sum2);
  g.in = at16(p.e.in);
  const float* part = a.part + split * a.plane + p.part0 + at;
  g.part = make_rsrc(part, a.ksplit > 1 ? 2u * bytes : 0u);
  g.part2 = make_rsrc(part + (int64_t)p.M * p.N, a.ksplit > 1 && two ? 2u * bytes : 0u);
  g.bias = make_rsrc(p.e.bias, p.e.bias != nullptr ? (uint32_t)p.N * 2u : 0u);
  g.keep = p.e.sum != nullptr;
  return g;
}
__device__ __forceinline__ void dg_st8(__amdgpu_buffer_rsrc_t r, int o, const float v[8]) {
  __builtin_amdgcn_raw_buffer_store_b128(dg_pack8(v), r, 2 * o, 0, 0);
}
__device__ __forceinline__ void dg_st8_f32(__amdgpu_buffer_rsrc_t r, int o, const float v[8]) {
#pragma unroll
  for (int k = 0; k < 8; k += 4)
    __builtin_amdgcn_raw_buffer_store_b128(u32x4_t{__float_as_uint(v[k]), __float_as_uint(v[k + 1]),
                                                   __float_as_uint(v[k + 2]), __float_as_uint(v[k + 3])},
                                           r, 4 * (o + k), 0, 0);
}

// d/dx gelu_tanh = s + x s (1 - s) 2 u', s = 1 / (1 + exp(-2 u)),
// u' = sqrt(2/pi) (1 + 3 0.044715 x^2); beyond |x| = 12 it is 0 or 1 (the
// comparisons leave a NaN as it is).
__device__ __forceinline__ void gelu_tanh_and_slope(float x, float* act, float* slope) {
  const float xc = x < -12.f ? -12.f : (x > 12.f ? 12.f : x);
  const float x2 = xc * xc;
  const float u = 0.7978845608028654f * xc * (1.0f + 0.044715f * x2);
  const float s = __fdividef(1.0f, 1.0f + __expf(-2.0f * u));
  *act = x * s;
  *slope = s + xc * s * (1.0f - s) * 1.5957691216057308f * (1.0f + 0.134145f * x2);
}
// gelu_erf = x Phi(x) and its slope Phi(x) + x phi(x), with the normal tail
// Q(|x|) = exp(-x^2 / 2) t P(t), t = 1 / (1 + 0.3 |x|).  P, of degree seven, is
// this file's own least-maximum fit of exp(x^2 / 2) Q(x) / t over 0 <= x <= 14:
// off by 1.5e-7 of itself in exact arithmetic and 6.5e-7 in fp32, the tail then by
// 1.2e-5 at most (the exponential's argument, rounded, at |x| = 13): far below
// a rounding to bf16, 3.9e-3.  A product of 2049 rows of 2816 takes 6 us longer
// with it than without an activation; erff and an exponential of their own, 16.
__device__ __forceinline__ void gelu_erf_and_slope(float x, float* act, float* slope) {
  const float e = __expf(-0.5f * x * x);
  const float t = __fdividef(1.0f, 1.0f + 0.3f * fabsf(x));
  float P = 0.0356754129f;
  P = __builtin_fmaf(P, t, -0.157205828f);
  P = __builtin_fmaf(P, t, 0.206358366f);
  P = __builtin_fmaf(P, t, -0.0536882205f);
  P = __builtin_fmaf(P, t, 0.128564095f);
  P = __builtin_fmaf(P, t, 0.0999127325f);
  P = __builtin_fmaf(P, t, 0.12075408f);
  P = __builtin_fmaf(P, t, 0.11962929f);
  const float q = t * P * e;
  const float cdf = x < 0.f ? q : 1.0f - q;
  *act = x * cdf;
  *slope = cdf + x * (0.3989422804014327f * e);
}

// what the epilogue reads at element o, column n: in, or sum and sum2; the bias
struct DgIn {
  u32x4_t v[4], bias;
};
template <int EPI>
__device__ __forceinline__ DgIn dg_fetch(const DgTarget& g, int o) {
  DgIn r;
  if (EPI == kDgGateUpBack) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      r.v[k] = buf_ld16(g.sum, 4 * o, 16 * k);
      r.v[2 + k] = buf_ld16(g.sum2, 4 * o, 16 * k);
    }
  } else if (EPI == kDgBiasResidual) {
    r.v[0] = buf_ld16(g.in, 2 * o, 0);
  } else if (EPI == kDgGeluBack) {
#pragma unroll
    for (int k = 0; k < 2; ++k) r.v[k] = buf_ld16(g.sum, 4 * o, 16 * k);
  }
  return r;
}
// the bias of columns n .. n + 7 (zeros past the problem)
template <int EPI>
__device__ __forceinline__ u32x4_t dg_bias(const DgTarget& g, int n) {
  return EPI == kDgBiasGelu || EPI == kDgBiasResidual ? buf_ld16(g.bias, 2 * n, 0) : u32x4_t{0u, 0u, 0u, 0u};
}

// v: the sums (v2: kDgGateUp's up sums) of the target's elements o .. o + 7
template <int EPI>
__device__ __forceinline__ void dg_finish(const DgTarget& g, int o, const float v[8], const float v2[8],
                                          const DgIn& in) {
  float r[8], s[8];
  if constexpr (EPI == kDgPlain) {
    dg_st8(g.out, o, v);
  } else if constexpr (EPI == kDgGateUp) {
    // h = gelu_tanh(a) b from the sums themselves, rounded once.  The backward
    // pass gets them as they are: rounded, they would cost its gradients as
    // much as da's and db's own rounding (relative error against 64 bits of dx,
    // dgate and dup 3.0e-3 instead of 2.4e-3).
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = gelu_tanh_f32(v[i]) * v2[i];
    dg_st8(g.out, o, r);
    if (g.keep) {
      dg_st8_f32(g.sum, o, v);
      dg_st8_f32(g.sum2, o, v2);
    }
  } else if constexpr (EPI == kDgGateUpBack) {
    const uint32_t a[8] = {in.v[0].x, in.v[0].y, in.v[0].z, in.v[0].w, in.v[1].x, in.v[1].y, in.v[1].z, in.v[1].w};
    const uint32_t b[8] = {in.v[2].x, in.v[2].y, in.v[2].z, in.v[2].w, in.v[3].x, in.v[3].y, in.v[3].z, in.v[3].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float act, slope;
      gelu_tanh_and_slope(__uint_as_float(a[i]), &act, &slope);
      r[i] = v[i] * __uint_as_float(b[i]) * slope;
      s[i] = v[i] * act;
    }
    dg_st8(g.out, o, r);
    dg_st8(g.out2, o, s);
  } else if constexpr (EPI == kDgBiasGelu) {
    dg_unpack8(in.bias, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float slope;
      s[i] += v[i];
      gelu_erf_and_slope(s[i], &r[i], &slope);
    }
    dg_st8(g.out, o, r);
    dg_st8_f32(g.sum, o, s);
  } else if constexpr (EPI == kDgBiasResidual) {
    float b[8];
    dg_unpack8(in.bias, b);
    dg_unpack8(in.v[0], s);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = s[i] + (v[i] + b[i]);
    dg_st8_f32(g.sum, o, r);
  } else if constexpr (EPI == kDgGeluBack) {
    const uint32_t z[8] = {in.v[0].x, in.v[0].y, in.v[0].z, in.v[0].w, in.v[1].x, in.v[1].y, in.v[1].z, in.v[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float act, slope;
      gelu_erf_and_slope(__uint_as_float(z[i]), &act, &slope);
      r[i] = v[i] * slope;
    }
    dg_st8(g.out, o, r);
  } else if constexpr (EPI == kDgSums) {
    dg_st8_f32(g.sum, o, v);
  }
}

// the workgroup's item: every XCD (workgroups go round robin) has a run of
// consecutive ones; -1 past them
__device__ __forceinline__ int dg_item(int total) {
  const int per = (total + 7) >> 3, x = (int)(blockIdx.x & 7), i = (int)(blockIdx.x >> 3);
  return i < per && x * per + i < total ? x * per + i : -1;
}

template <int LAYOUT, int EPI, int MI, int NI, int KG>
__global__ __launch_bounds__(KG * kDgThreads, MI * NI > 36 ? 1 : KG > 2 ? KG : 2) void k_gemm_dense(DgArgs a) {
  constexpr bool AC = LAYOUT == kDgTN, BC = LAYOUT != kDgNT;
  constexpr bool GU = EPI == kDgGateUp;
  constexpr bool kPairs = dg_pairs(LAYOUT);
  using OA = DgOperand<AC, false, MI, kPairs>;
  using OB = DgOperand<BC, GU, NI, kPairs>;
  constexpr int kSlot = dg_slot_bytes(LAYOUT, MI, NI);
  static_assert(kSlot == OA::kBytes + OB::kBytes, "a slot's operands");
  constexpr int kSlots = dg_slots(LAYOUT, MI, NI, KG);
  constexpr int kLoads = OA::kLoads + OB::kLoads;
  constexpr int BM = dg_bm(MI), BN = dg_bn(EPI, NI);
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
  const int group = KG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
  unsigned char* const ring = smem + group * kSlots * kSlot;

  // the tile: kDgGroupM row tiles run with each column tile
  int item = dg_item(a.tiles * a.ksplit);
  if (item < 0) return;
  const int split = item / a.tiles;
  item -= split * a.tiles;
  int pi = 0;
  while (pi + 1 < a.nprob && item >= a.prob[pi + 1].tile0) ++pi;
  const DgProblem& p = a.prob[pi];
  item -= p.tile0;
  const int n_mt = (p.M + BM - 1) / BM, n_nt = (p.N + BN - 1) / BN;
  const int grp = item / (kDgGroupM * n_nt);
  const int rem = item - grp * kDgGroupM * n_nt;
  const int gm = min(kDgGroupM, n_mt - grp * kDgGroupM);
  const int nt = rem / gm;
  const int m0 = (grp * kDgGroupM + rem - nt * gm) * BM, n0 = nt * BN;
  // the group's stages; every group runs as many (those past its range multiply
  // the zeros that empty descriptors give)
  constexpr int kStep = kPairs ? 2 : 1;
  const int per = (a.nk + kStep * a.ksplit * KG - 1) / (kStep * a.ksplit * KG) * kStep;
  // what is loaded next, kSlots ahead of the multiplication: stage t of the
  // operands (their values here: the loop reads no arguments)
  struct Feed {
    const uint16_t *A, *A2, *B, *B2;
    int M, N, lda, ldb, t, end;
  };
  Feed f{p.A, p.A2, p.B, p.B2, p.M, p.N, p.lda, p.ldb, (split * KG + group) * per, 0};
  f.end = min(a.nk, f.t + per);
  OA oa;
  OB ob;
  oa.init(m0, f.M, f.lda, wave);
  ob.init(n0, f.N, f.ldb, wave);
  oa.init_frag(wave >> 1);
  ob.init_frag(wave & 1);

  // Where the next stage's loads come from.  The descriptors are empty past the
  // range; cols: they start at the stage's first k and end with row K - 1, so
  // that rows past K read as zero.  Rows: stages of the second pair (t >= nk1)
  // follow the first's.
  struct Src {
    __amdgpu_buffer_rsrc_t a, b, b2;
    int off;
    int skip;  // pairs: a lane's chunk is past K (a last pair of one stage)
  };
  const bool second = kPairs && (((lane >> 2) ^ wave) & 1) != 0;  // its chunk is of a pair's second stage
  auto source = [&] {
    const bool two = LAYOUT == kDgNN && f.t >= a.nk1;
    const int tt = two ? f.t - a.nk1 : f.t;
    const bool any = f.t < f.end;
    const int left = min(kDgKT, a.K - tt * kDgKT);
    const uint16_t* pa = two ? f.A2 : f.A;
    const uint16_t* pb = two ? f.B2 : f.B;
    Src r;
    r.a = AC ? make_rsrc(pa + (int64_t)tt * kDgKT * f.lda + m0, any ? (uint32_t)(left * f.lda - m0) * 2u : 0u)
             : make_rsrc(pa + (int64_t)m0 * f.lda, any ? (uint32_t)(min(f.M - m0, BM) * f.lda) * 2u : 0u);
    const uint32_t bbytes = (uint32_t)(min(f.N - n0, BN) * f.ldb) * 2u;
    r.b = BC ? make_rsrc(pb + (int64_t)tt * kDgKT * f.ldb + n0, any ? (uint32_t)(left * f.ldb - n0) * 2u : 0u)
             : make_rsrc(pb + (int64_t)n0 * f.ldb, any ? bbytes : 0u);
    r.b2 = GU ? make_rsrc(f.B2 + (int64_t)n0 * f.ldb, any ? bbytes : 0u) : r.b;
    r.off = tt * (kDgKT * 2);
    r.skip = kPairs && second && f.t + 1 >= a.nk ? kDgOut : 0;
    f.t += kStep;
    return r;
  };
  // load j of the wavefront's kLoads into a slot
  auto issue = [&](const Src& r, unsigned char* slot, int j) {
    if (j < OA::kLoads) {
      px_dma16(r.a, oa.voff[j] + r.skip, AC ? 0 : r.off, slot + (wave + 4 * j) * 1024);
    } else {
      const int i = j - OA::kLoads;
      if (GU && OB::second(i, wave))
        px_dma16(r.b2, ob.voff[i] + r.skip, r.off, slot + OA::kBytes + (wave + 4 * i) * 1024);
      else
        px_dma16(r.b, ob.voff[i] + r.skip, BC ? 0 : r.off, slot + OA::kBytes + (wave + 4 * i) * 1024);
    }
  };

  // Accumulators past what the vector registers hold live in the accumulation
  // registers.  Named so before and after the loop, each keeps one place in
  // it; otherwise the compiler moves up to 200 of them around per stage.
  f32x4_t acc[MI][NI];
  constexpr bool kAccRegs = MI * NI > 36;
  auto pin = [&] {
    if constexpr (kAccRegs) {
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n) asm volatile("" : "+a"(acc[m][n]));
    }
  };
  constexpr int NO = GU ? NI / 2 : NI;  // 16-column tiles of results per wavefront
  constexpr int kPlanes = GU ? 2 : 1;
  constexpr int kIter = (2 * 16 * NO + 63) / 64;
  // column fragments twice where there is room: those of the next stage are
  // then read all along a stage
  constexpr int kB = kAccRegs ? 2 : 1;
  u32x4_t fa[MI], fb[kB][NI];

#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    const Src r = source();
#pragma unroll
    for (int j = 0; j < kLoads; ++j) issue(r, ring + s * kSlot, j);
  }
  dg_wait_vm<(kSlots - 1) * kLoads>();
  px_barrier();
#pragma unroll
  for (int n = 0; n < NI; ++n) fb[0][n] = ob.frag(ring + OA::kBytes, n, 0);
#pragma unroll
  for (int m = 0; m < MI; ++m) fa[m] = oa.frag(ring, m, 0);

  // Stage t, its fragments at hand.  Every fragment register takes its fragment
  // of stage t + 1 after its last MFMA.  In a slot's last stage the wavefronts
  // meet after the first row of fragments' MFMAs (the next slot has landed, this
  // one is read), then the slot is refilled, kSlots ahead.  Reads and loads go
  // one by one between the MFMAs: one after every second keeps the matrix unit
  // fed.
  int slot = 0;
  auto stage = [&](auto cur_) {
    constexpr int cur = kB == 2 ? decltype(cur_)::value : 0, nxt = kB == 2 ? cur ^ 1 : 0;
    constexpr int at = kPairs ? decltype(cur_)::value : 0;  // the stage of its slot
    constexpr bool kMeet = at == kStep - 1;
    constexpr int kIssue = kMeet ? kLoads : 0, kNext = kMeet ? 0 : at + 1;
    const int ns = kMeet ? (slot == kSlots - 1 ? 0 : slot + 1) : slot;
    unsigned char* refill = ring + slot * kSlot;
    const unsigned char* st = ring + ns * kSlot;
    Src src;
    if constexpr (kMeet) src = source();
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[0][n] = mfma16(fb[cur][n], fa[0], acc[0][n]);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (kMeet) {
      dg_wait_vm<(kSlots - 2) * kLoads>();
      px_barrier();
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (kB == 2) {
      // operation o of the row m: its MFMAs are done one ahead
      constexpr int R = MI - 1;
#pragma unroll
      for (int m = 1; m < MI; ++m) {
        // this row's: fa[m - 1], then column fragments and loads by turns
        const int b0 = (m - 1) * NI / R, b1 = m * NI / R, l0 = (m - 1) * kIssue / R, l1 = m * kIssue / R;
        int done = 0;
#pragma unroll
        for (int n = 0; n < NI; ++n) {
          acc[m][n] = mfma16(fb[cur][n], fa[m], acc[m][n]);
          if (n % 2 == 0 || NI < 6) {
            if (done == 0) {
              fa[m - 1] = oa.frag(st, m - 1, kNext);
            } else {
              const int k = done - 1;
              if (k < b1 - b0)
                fb[nxt][b0 + k] = ob.frag(st + OA::kBytes, b0 + k, kNext);
              else if (k - (b1 - b0) < l1 - l0)
                issue(src, refill, l0 + k - (b1 - b0));
            }
            ++done;
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        // what did not fit
#pragma unroll
        for (int k = done - 1; k < (b1 - b0) + (l1 - l0); ++k) {
          if (k < b1 - b0)
            fb[nxt][b0 + k] = ob.frag(st + OA::kBytes, b0 + k, kNext);
          else
            issue(src, refill, l0 + k - (b1 - b0));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      fa[MI - 1] = oa.frag(st, MI - 1, kNext);
    } else {
      if (MI > 2) fa[0] = oa.frag(st, 0, kNext);
#pragma unroll
      for (int m = 1; m < MI - 2; ++m) {
#pragma unroll
        for (int n = 0; n < NI; ++n) acc[m][n] = mfma16(fb[0][n], fa[m], acc[m][n]);
        fa[m] = oa.frag(st, m, kNext);
#pragma unroll
        for (int j = (m - 1) * kIssue / (MI > 3 ? MI - 3 : 1); j < m * kIssue / (MI > 3 ? MI - 3 : 1); ++j)
          issue(src, refill, j);
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (MI <= 3) {
#pragma unroll
        for (int j = 0; j < kIssue; ++j) issue(src, refill, j);
      }
      // the last two rows column by column, so that a column's fragment has
      // 2 (NI - 1) MFMAs to arrive
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        if (MI > 2) acc[MI - 2][n] = mfma16(fb[0][n], fa[MI - 2], acc[MI - 2][n]);
        acc[MI - 1][n] = mfma16(fb[0][n], fa[MI - 1], acc[MI - 1][n]);
        fb[0][n] = ob.frag(st + OA::kBytes, n, kNext);
        __builtin_amdgcn_sched_barrier(0);
      }
      fa[MI - 2] = oa.frag(st, MI - 2, kNext);
      fa[MI - 1] = oa.frag(st, MI - 1, kNext);
    }
    slot = ns;
  };

#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  pin();
  if constexpr (kB == 2 || kPairs) {
    for (int t = 0; t < per; t += 2) {
      stage(std::integral_constant<int, 0>{});
      if (kPairs || t + 1 < per) stage(std::integral_constant<int, 1>{});
    }
  } else {
    for (int t = 0; t < per; ++t) stage(std::integral_constant<int, 0>{});
  }
  pin();
  dg_wait_vm<0>();  // no load may land in what the ring's place holds next,
  px_barrier();     // and every wavefront is past its reads of the ring
  if constexpr (KG > 1) {
    // the groups' sums, added in order
    f32x4_t* const sums = reinterpret_cast<f32x4_t*>(smem) + wave * MI * NI * 64 + lane;
    if (group > 0) {
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n) sums[((group - 1) * 4 * MI * NI + m * NI + n) * 64] = acc[m][n];
    }
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int g = 1; g < KG; ++g)
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n) acc[m][n] += sums[((g - 1) * 4 * MI * NI + m * NI + n) * 64];
  }

  // Epilogue, 16 rows of the wavefront at a time: lane l holds columns
  // 4 (l / 16) .. + 3 of row l % 16 of each 16 x 16 tile; through the
  // wavefront's own part of the LDS it gets eight consecutive columns of a row,
  // so that every load and store is 16 bytes per lane and whole rows of the
  // wavefront's columns (8 bytes in 32-byte pieces took half as long again).
  constexpr int kPitch = dg_epi_pitch(NO);
  constexpr int kSums = (KG - 1) * 4 * MI * NI * 1024;
  static_assert(kSums + 4 * kPlanes * 16 * kPitch * 4 <= KG * kSlots * kSlot, "the epilogue's rows fit in the ring");
  float* const rows = reinterpret_cast<float*>(smem + kSums) + wave * kPlanes * 16 * kPitch;
  const int r0 = m0 + 16 * MI * (wave >> 1), c0 = n0 + 16 * NO * (wave & 1);
  const DgTarget g = dg_target(a, p, split, r0, 16 * MI, GU);
  // What it reads is asked for some steps of 16 rows before it is needed: a step
  // by itself would wait for memory.  Four vectors per element (kDgGateUpBack)
  // leave registers for one step ahead, once a step's sums are in LDS (8192 rows
  // 2816 -> 2112 139 to 134 us), and in 4 x 8 tiles for none.  Two (kDgGeluBack)
  // leave them for one step in the tiles that fill the vector registers.
  constexpr bool kFull = MI * NI > 24 && !kAccRegs;
  constexpr int kAhead = EPI == kDgGateUpBack ? (kIter > 3 && !kAccRegs ? 0 : 1) : EPI == kDgGeluBack && kFull ? 1 : 3;
  constexpr bool kLate = kAhead == 1;
  DgIn in[MI][kIter];
  int o[MI][kIter];
  u32x4_t bias[kIter];
  auto fetch = [&](int m) {
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int idx = lane + 64 * i, col = c0 + 8 * (idx % (2 * NO));
      // element of the target; past it for lanes past the tile and columns past the problem
      o[m][i] = idx < 32 * NO && col < p.N ? (16 * m + idx / (2 * NO)) * p.N + col : kDgOut;
      in[m][i] = dg_fetch<EPI>(g, o[m][i]);
    }
  };
#pragma unroll
  for (int i = 0; i < kIter; ++i) bias[i] = dg_bias<EPI>(g, c0 + 8 * ((lane + 64 * i) % (2 * NO)));
#pragma unroll
  for (int m = 0; m < kAhead && m < MI; ++m) fetch(m);
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    if (!kLate && m + kAhead < MI) fetch(m + kAhead);
#pragma unroll
    for (int n = 0; n < NO; ++n) {
      float* q = rows + (lane & 15) * kPitch + 16 * n + 4 * (lane >> 4);
      *reinterpret_cast<f32x4_t*>(q) = acc[m][n];
      if (GU) *reinterpret_cast<f32x4_t*>(q + 16 * kPitch) = acc[m][GU ? n + NO : n];
    }
    if (kLate && m + kAhead < MI) fetch(m + kAhead);
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int idx = min(lane + 64 * i, 32 * NO - 1);
      const float* q = rows + idx / (2 * NO) * kPitch + 8 * (idx % (2 * NO));
      float v[8], v2[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] = q[k];
        v2[k] = GU ? q[16 * kPitch + k] : 0.f;
      }
      if (a.ksplit > 1) {
        dg_st8_f32(g.part, o[m][i], v);
        if (GU) dg_st8_f32(g.part2, o[m][i], v2);
      } else {
        in[m][i].bias = bias[i];
        dg_finish<EPI>(g, o[m][i], v, v2, in[m][i]);
      }
    }
  }
}

// The sums of a split launch: the splits' partial sums in order, then the
// epilogue; a thread has eight columns of one row.
template <int EPI>
__global__ __launch_bounds__(256) void k_gemm_dense_join(DgArgs a) {
  const DgProblem& p = a.prob[blockIdx.y];
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)p.M * p.N / 8) return;
  const int row = (int)(8 * i / p.N), n = (int)(8 * i - (int64_t)row * p.N);
  // from the workgroup's first row on: some 2048 elements of few rows, or of one
  const int row0 = (int)((int64_t)blockIdx.x * 2048 / p.N);
  const DgTarget g = dg_target(a, p, 0, row0, 256, false);
  const int o = (row - row0) * p.N + n;
  DgIn in = dg_fetch<EPI>(g, o);
  in.bias = dg_bias<EPI>(g, n);
  const float* q = a.part + p.part0 + 8 * i;
  float v[8], v2[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = v2[k] = 0.f;
#pragma unroll 4
  for (int s = 0; s < a.ksplit; ++s) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] += q[s * a.plane + k];
      if (EPI == kDgGateUp) v2[k] += q[s * a.plane + (int64_t)p.M * p.N + k];
    }
  }
  dg_finish<EPI>(g, o, v, v2, in);
}

template <int LAYOUT, int EPI, int MI, int NI, int KG>
hipError_t dg_launch(const DgArgs& a, hipStream_t s) {
  constexpr int lds = KG * dg_slots(LAYOUT, MI, NI, KG) * dg_slot_bytes(LAYOUT, MI, NI);
  static_assert(lds <= 160 * 1024, "LDS of a CU");
  const int64_t groups = ((int64_t)a.tiles * a.ksplit + 7) / 8;  // of eight workgroups, one per XCD
  hipLaunchKernelGGL((k_gemm_dense<LAYOUT, EPI, MI, NI, KG>), dim3((unsigned)(8 * groups)), dim3(KG * kDgThreads), lds,
                     s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.ksplit == 1) return e;
  int64_t most = 0;
  for (int i = 0; i < a.nprob; ++i) most = std::max(most, (int64_t)a.prob[i].M * a.prob[i].N / 8);
  hipLaunchKernelGGL(k_gemm_dense_join<EPI>, dim3((unsigned)((most + 255) / 256), a.nprob), dim3(256), 0, s, a);
  return hipGetLastError();
}

// the launch with the tile that `a` was planned for
template <int LAYOUT, int EPI>
hipError_t dg_launch_tile(const DgArgs& a, hipStream_t s) {
#define W4A16_DG(MI_, NI_, KG_, OCC_, ALONE_, EACH_) \
  if (a.mi == MI_ && a.ni == NI_ && a.kg == KG_) return dg_launch<LAYOUT, EPI, MI_, NI_, KG_>(a, s);
  if constexpr (LAYOUT == kDgNT) {
    W4A16_DG_TILES_NT(W4A16_DG)
  } else if constexpr (LAYOUT == kDgNN) {
    W4A16_DG_TILES_NN(W4A16_DG)
  } else {
    W4A16_DG_TILES_TN(W4A16_DG)
  }
#undef W4A16_DG
  return hipErrorInvalidValue;
}

}  // namespace w4a16
