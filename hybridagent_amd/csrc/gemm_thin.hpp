// Dense bf16 products of few rows: the weights' stream.
//
//   kDgNT  y = x W^T,  kDgNN  dx = dy W   (gemm_dense.hpp's problems and epilogues)
//
// A workgroup owns 16 or 32 columns (gate/up: 16 gate columns and their up
// columns) of up to 16 MT rows; its wavefronts, eight where their slots fit,
// split K, each with a ring of LDS slots of its own, so that nothing in the
// loop waits for another wavefront.  A stage is 64 k, by direct loads.  The
// partial tiles are added in wavefront order in LDS and finished there: one
// launch, where a product split over workgroups needs a second one to add its
// planes.
//
// Bound: what a CU takes from the caches, some 130 bytes per ns, if whole
// 128-byte lines are asked for: a line that comes in two stages of 64 bytes
// each has left the L1 between them and comes twice (2816 -> 2816, stages of
// 32 / 64 k: 16 rows 8.0/6.3 us, 32 9.6/7.3, 64 11.9/8.9).  dy W's weights come
// in 64-byte pieces, one half of a line to each of two workgroups.  Then
// latency: the first stage, the reduction, the launch.
#pragma once
#include "gemm_dense.hpp"

namespace w4a16 {

// wavefronts: eight with two slots each at least, else four (sixteen gained
// nothing: 1, 16, 32 rows of 2816 -> 2816 5.4, 6.2, 7.9 us with eight, 5.9, 6.6, 8.3)
constexpr int thin_waves(int mt, int nw) { return mt + nw > 5 ? 4 : 8; }
constexpr int kThinKT = 64;  // k per stage
// slots per wavefront that fit in a CU's LDS
constexpr int thin_stages(int mt, int nw) { return 80 / thin_waves(mt, nw) / (mt + nw); }

template <int LAYOUT, int EPI, int MT, int NW>
__global__ __launch_bounds__(64 * thin_waves(MT, NW)) void k_gemm_thin(DgArgs a) {
  constexpr int kThinWaves = thin_waves(MT, NW);
  constexpr bool COLS = LAYOUT == kDgNN;
  constexpr bool GU = EPI == kDgGateUp;
  static_assert((!COLS && !GU) || NW == 2, "32 columns; gate and up columns");
  constexpr int kStages = thin_stages(MT, NW);
  constexpr int kW = 2 * NW, kLoads = kW + 2 * MT;
  constexpr int kStage = 1024 * kLoads;
  constexpr int BN = GU ? 16 : 16 * NW;
  static_assert(kStages >= 2 && kThinWaves * kStages * kStage <= 160 * 1024, "LDS of a CU");
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const DgProblem& p = a.prob[0];
  const int M = p.M, N = p.N, lda = p.lda, ldb = p.ldb;
  // neighbouring columns on one XCD: in [k][n] rows they share cache lines
  const int n_nt = (N + BN - 1) / BN, item = dg_item(n_nt);
  if (item < 0) return;
  const int n0 = item * BN, m0 = blockIdx.y * 16 * MT;
  // stages of the first pair, and of both; the wavefront's
  const int n1 = (a.K + kThinKT - 1) / kThinKT, nk = COLS && p.A2 != nullptr ? 2 * n1 : n1;
  const int per = (nk + kThinWaves - 1) / kThinWaves;
  const int t0 = wave * per, t1 = min(nk, t0 + per);
  unsigned char* const ring = smem + wave * kStages * kStage;

  // Rows format: load j brings eight rows, lane l the 16-byte chunk (l % 8) ^
  // swizzle of row 8 j + l / 8, so that the 16 lanes that a fragment's read
  // serves at once cover the banks.  Rows past the problem repeat its last.
  // A last stage of 32 k: its chunks 4 .. 7 (lanes of bit 2 unlike j) are past it.
  const auto chunk = [&](int j) { return (lane & 7) ^ (((8 * j + (lane >> 3)) >> 1) & 7); };
  int wv[kW], av[2 * MT], wf[2];
#pragma unroll
  for (int j = 0; j < kW; ++j) {
    if constexpr (COLS) {
      // two blocks of [32 k][32 columns], 64 bytes a row: load j brings k 16 j ..,
      // lane l row l / 4.  The halves of a row change places where bit 3 of k is
      // set: a transposing read's 32 lanes take rows 0 .. 3 and 8 .. 11 (+ 4).
      const int k = 16 * j + (lane >> 2);
      wv[j] = k * ldb * 2 + 2 * min(8 * ((lane & 3) ^ (((k >> 3) & 1) << 1)), N - n0 - 8);
    } else {
      const int r = (GU ? 8 * (j & 1) : 8 * j) + (lane >> 3);
      wv[j] = min(r, N - n0 - 1) * ldb * 2 + 16 * chunk(j);
    }
  }
#pragma unroll
  for (int j = 0; j < 2 * MT; ++j) av[j] = min(8 * j + (lane >> 3), M - m0 - 1) * lda * 2 + 16 * chunk(j);
  const int rf = (lane & 15) * 128 + 16 * ((lane >> 4) ^ ((lane >> 1) & 7));  // the second 32 k: ^ 64
#pragma unroll
  for (int n = 0; n < 2; ++n)
    wf[n] = (8 * (lane >> 4) + ((lane & 15) >> 2)) * 64 + 32 * (n ^ ((lane >> 4) & 1)) + 8 * (lane & 3);

  auto issue = [&](int t, unsigned char* st) {
    const bool two = COLS && t >= n1;
    const int k = (two ? t - n1 : t) * kThinKT;
    const bool any = t < t1;
    const int left = min(kThinKT, a.K - k);
    const int past = left < kThinKT ? kDgOut : 0;
    const int skip[2] = {lane & 4 ? past : 0, lane & 4 ? 0 : past};  // even and odd j
    const uint16_t* pa = two ? p.A2 : p.A;
    const uint16_t* pb = two ? p.B2 : p.B;
    const auto ra = make_rsrc(pa + (int64_t)m0 * lda, any ? (uint32_t)(min(M - m0, 16 * MT) * lda) * 2u : 0u);
    const auto rb = COLS ? make_rsrc(pb + (int64_t)k * ldb + n0, any ? (uint32_t)(left * ldb - n0) * 2u : 0u)
                         : make_rsrc(pb + (int64_t)n0 * ldb, any ? (uint32_t)(min(N - n0, BN) * ldb) * 2u : 0u);
    const auto rb2 = GU ? make_rsrc(p.B2 + (int64_t)n0 * ldb, any ? (uint32_t)(min(N - n0, 16) * ldb) * 2u : 0u) : rb;
#pragma unroll
    for (int j = 0; j < kW; ++j)
      px_dma16(GU && j >= 2 ? rb2 : rb, COLS ? wv[j] : wv[j] + skip[j & 1], COLS ? 0 : 2 * k, st + 1024 * j);
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j) px_dma16(ra, av[j] + skip[j & 1], 2 * k, st + 1024 * (kW + j));
  };

  // what the epilogue reads: asked for first, a memory's latency before its use
  constexpr int NC = BN / 8;  // 8-column pieces of a row
  const int row = threadIdx.x / NC, c = threadIdx.x % NC;
  const DgTarget g = dg_target(a, p, 0, m0, 16 * MT, false);
  const int o = row < 16 * MT && n0 + 8 * c < N ? row * N + n0 + 8 * c : kDgOut;
  DgIn in = dg_fetch<EPI>(g, o);
  in.bias = dg_bias<EPI>(g, n0 + 8 * c);
  f32x4_t acc[MT][NW];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NW; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < kStages; ++s) issue(t0 + s, ring + s * kStage);
  int slot = 0;
  for (int t = t0; t < t1; ++t) {
    unsigned char* st = ring + slot * kStage;
    __builtin_amdgcn_sched_barrier(0);
    dg_wait_vm<(kStages - 1) * kLoads>();  // the stage has landed
    __builtin_amdgcn_sched_barrier(0);
    u32x4_t fb[2][NW], fa[2][MT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int n = 0; n < NW; ++n) {
        if constexpr (COLS) {
          const unsigned char* q = st + 2048 * h + wf[n];
          const bf16x4_t lo = dg_tr_read((lds_bf16x4_t*)q);
          const bf16x4_t hi = dg_tr_read((lds_bf16x4_t*)(q + 256));
          const bf16x8_t v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          fb[h][n] = __builtin_bit_cast(u32x4_t, v);
        } else {
          fb[h][n] = *reinterpret_cast<const u32x4_t*>(st + 2048 * n + (rf ^ (64 * h)));
        }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
        fa[h][i] = *reinterpret_cast<const u32x4_t*>(st + 1024 * kW + 2048 * i + (rf ^ (64 * h)));
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the slot is read
    __builtin_amdgcn_sched_barrier(0);
    issue(t + kStages, st);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NW; ++n) acc[i][n] = mfma16(fb[h][n], fa[h][i], acc[i][n]);
    slot = slot == kStages - 1 ? 0 : slot + 1;
  }
  dg_wait_vm<0>();
  px_barrier();
  // partial tiles [wavefront][16 MT rows][16 NW columns]
  constexpr int kPitch = 16 * NW + 4;
  float* const red = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NW; ++j)
      *reinterpret_cast<f32x4_t*>(red + ((wave * MT + i) * 16 + (lane & 15)) * kPitch + 16 * j + 4 * (lane >> 4)) =
          acc[i][j];
  __syncthreads();
  if (row >= 16 * MT || m0 + row >= M || n0 + 8 * c >= N) return;
  float v[8], v2[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = v2[k] = 0.f;
#pragma unroll
  for (int w = 0; w < kThinWaves; ++w) {
    const float* q = red + (w * 16 * MT + row) * kPitch + 8 * c;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] += q[k];
      if (GU) v2[k] += q[16 + k];
    }
  }
  dg_finish<EPI>(g, o, v, v2, in);
}

template <int LAYOUT, int EPI, int MT, int NW>
hipError_t thin_start(const DgArgs& a, hipStream_t s) {
  constexpr int bn = EPI == kDgGateUp ? 16 : 16 * NW;
  hipLaunchKernelGGL((k_gemm_thin<LAYOUT, EPI, MT, NW>),
                     dim3(8 * (((a.prob[0].N + bn - 1) / bn + 7) / 8), (a.prob[0].M + 16 * MT - 1) / (16 * MT)),
                     dim3(64 * thin_waves(MT, NW)), thin_waves(MT, NW) * thin_stages(MT, NW) * 2048 * (NW + MT), s, a);
  return hipGetLastError();
}

template <int LAYOUT, int EPI>
hipError_t thin_launch(const DgArgs& a, hipStream_t s) {
  const int M = a.prob[0].M, N = a.prob[0].N;
  // One round of workgroups (one a CU) decides.  16 columns each while those
  // are no more than the CUs (1, 16, 32 rows, 32 / 16 columns: 2816 -> 2816
  // 5.8/5.6, 6.3/5.7, 7.3/6.5 us, 2816 -> 5632 7.3/9.7, 7.4/10.1, 8.3/11.4);
  // dy W always 32, whose pieces of rows would be 32 bytes (9.5/10.3 us).  Of
  // more than 32 rows each half by itself while both fit (64 rows, halves /
  // together: 2816 -> 2816 7.3/8.9, 2816 -> 8192 18.2/11.7).
  const int cus = device_cus();
  if constexpr (EPI != kDgGateUp && LAYOUT == kDgNT) {
    if (M <= 32 && (N + 15) / 16 <= cus)
      return M <= 16 ? thin_start<LAYOUT, EPI, 1, 1>(a, s) : thin_start<LAYOUT, EPI, 2, 1>(a, s);
  }
  const int bn = EPI == kDgGateUp ? 16 : 32;
  if (M <= 16) return thin_start<LAYOUT, EPI, 1, 2>(a, s);
  if (M <= 32 || 2 * ((N + bn - 1) / bn) <= cus) return thin_start<LAYOUT, EPI, 2, 2>(a, s);
  return thin_start<LAYOUT, EPI, 4, 2>(a, s);
}

}  // namespace w4a16
