// Dense bf16 products of few rows (M <= 64): the weights' stream.
//
//   kDgNT  y = x W^T,  kDgNN  dx = dy W   (gemm_dense.hpp's problems and epilogues)
//
// A workgroup of eight wavefronts owns 32 columns (gate/up: 16 gate columns
// and their up columns) of up to 16 MT rows; its wavefronts split K, each
// with a ring of LDS slots of its own, so that nothing in the loop waits for
// another wavefront.  A stage is 32 k: 2 KB of weights and MT KB of rows by
// direct loads, in gemm_dense.hpp's formats.  The eight partial tiles are
// added in wavefront order in LDS and finished there: one launch, where a
// product split over workgroups needs a second one to add its planes
// (2816 x 2816 at 32 rows: 10.3 us of two launches).
//
// Bound: the weights from memory, in practice latency (a wavefront's first
// stage, the reduction, the launch).
#pragma once
#include "gemm_dense.hpp"

namespace w4a16 {

constexpr int kThinWaves = 8;
constexpr int kThinThreads = 64 * kThinWaves;
// slots per wavefront that fit in a CU's LDS
constexpr int thin_stages(int mt) { return mt == 1 ? 6 : mt == 2 ? 4 : 3; }

template <int LAYOUT, int EPI, int MT>
__global__ __launch_bounds__(kThinThreads) void k_gemm_thin(DgArgs a) {
  constexpr bool COLS = LAYOUT == kDgNN;
  constexpr bool GU = EPI == kDgGateUp;
  constexpr int kStages = thin_stages(MT);
  constexpr int kStage = 2048 + 1024 * MT;
  constexpr int kLoads = 2 + MT;
  static_assert(kThinWaves * kStages * kStage <= 160 * 1024, "LDS of a CU");
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const DgProblem& p = a.prob[0];
  const int M = p.M, N = p.N, lda = p.lda, ldb = p.ldb;
  // neighbouring columns on one XCD: in [k][n] rows they share cache lines
  const int n_nt = (N + (GU ? 15 : 31)) / (GU ? 16 : 32), item = dg_item(n_nt);
  if (item < 0) return;
  const int n0 = item * (GU ? 16 : 32), m0 = blockIdx.y * 16 * MT;
  const int per = (a.nk + kThinWaves - 1) / kThinWaves;
  const int t0 = wave * per, t1 = min(a.nk, t0 + per);
  unsigned char* const ring = smem + wave * kStages * kStage;

  // sources: weight load j and row load i of a stage (rows and columns past the
  // problem repeat its last)
  int wv[2], av[MT], wf[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if constexpr (COLS) {
      // [32 k][32 columns], 64 bytes a row: load j brings k 16 j .., lane l row
      // l / 4.  The halves of a row change places where bit 3 of k is set: a
      // transposing read's 32 lanes take rows 0 .. 3 and 8 .. 11 (+ 4).
      const int k = 16 * j + (lane >> 2);
      const int chunk = (lane & 3) ^ (((k >> 3) & 1) << 1);
      wv[j] = k * ldb * 2 + 2 * min(8 * chunk, N - n0 - 8);
      const int kf = 8 * (lane >> 4) + ((lane & 15) >> 2);
      wf[j] = kf * 64 + 32 * (j ^ ((lane >> 4) & 1)) + 8 * (lane & 3);
    } else {
      const int r = (GU ? 0 : 16 * j) + (lane >> 2);
      const int chunk = (lane & 3) ^ dg_row_swz((lane >> 4) & 3);
      wv[j] = min(r, N - n0 - 1) * ldb * 2 + 16 * chunk;
      wf[j] = 1024 * j + (lane & 15) * 64 + 16 * ((lane >> 4) ^ dg_row_swz((lane >> 2) & 3));
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
    av[i] = min(16 * i + (lane >> 2), M - m0 - 1) * lda * 2 + 16 * ((lane & 3) ^ dg_row_swz((lane >> 4) & 3));
  const int af = (lane & 15) * 64 + 16 * ((lane >> 4) ^ dg_row_swz((lane >> 2) & 3));

  auto issue = [&](int t, unsigned char* st) {
    const bool two = COLS && t >= a.nk1;
    const int tt = two ? t - a.nk1 : t;
    const bool any = t < t1;
    const uint16_t* pa = two ? p.A2 : p.A;
    const uint16_t* pb = two ? p.B2 : p.B;
    const auto ra = make_rsrc(pa + (int64_t)m0 * lda, any ? (uint32_t)(min(M - m0, 16 * MT) * lda) * 2u : 0u);
    const auto rb = COLS ? make_rsrc(pb + (int64_t)tt * kDgKT * ldb + n0, any ? (uint32_t)(kDgKT * ldb - n0) * 2u : 0u)
                         : make_rsrc(pb + (int64_t)n0 * ldb, any ? (uint32_t)(min(N - n0, 32) * ldb) * 2u : 0u);
    const auto rb2 = GU ? make_rsrc(p.B2 + (int64_t)n0 * ldb, any ? (uint32_t)(min(N - n0, 16) * ldb) * 2u : 0u) : rb;
    const int off = tt * (kDgKT * 2);
    px_dma16(rb, wv[0], COLS ? 0 : off, st);
    px_dma16(rb2, wv[1], COLS ? 0 : off, st + 1024);
#pragma unroll
    for (int i = 0; i < MT; ++i) px_dma16(ra, av[i], off, st + 2048 + 1024 * i);
  };

  f32x4_t acc[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < kStages; ++s) issue(t0 + s, ring + s * kStage);
  int slot = 0;
  for (int t = t0; t < t1; ++t) {
    unsigned char* st = ring + slot * kStage;
    __builtin_amdgcn_sched_barrier(0);
    dg_wait_vm<(kStages - 1) * kLoads>();  // the stage has landed
    __builtin_amdgcn_sched_barrier(0);
    u32x4_t fb[2], fa[MT];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if constexpr (COLS) {
        const bf16x4_t lo = dg_tr_read((lds_bf16x4_t*)(st + wf[j]));
        const bf16x4_t hi = dg_tr_read((lds_bf16x4_t*)(st + wf[j] + 256));
        const bf16x8_t v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        fb[j] = __builtin_bit_cast(u32x4_t, v);
      } else {
        fb[j] = *reinterpret_cast<const u32x4_t*>(st + wf[j]);
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) fa[i] = *reinterpret_cast<const u32x4_t*>(st + 2048 + 1024 * i + af);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the slot is read
    __builtin_amdgcn_sched_barrier(0);
    issue(t + kStages, st);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = mfma16(fb[j], fa[i], acc[i][j]);
    slot = slot == kStages - 1 ? 0 : slot + 1;
  }
  dg_wait_vm<0>();
  px_barrier();
  // partial tiles [wavefront][16 MT rows][32 columns], rows 36 floats apart
  constexpr int kPitch = 36;
  float* const red = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      *reinterpret_cast<f32x4_t*>(red + ((wave * MT + i) * 16 + (lane & 15)) * kPitch + 16 * j + 4 * (lane >> 4)) =
          acc[i][j];
  __syncthreads();
  constexpr int NC = GU ? 2 : 4;  // 8-column pieces of a row
  const int row = threadIdx.x / NC, c = threadIdx.x % NC;
  if (row >= 16 * MT || m0 + row >= M || n0 + 8 * c >= N) return;
  const DgTarget g = dg_target(a, p, 0, m0, 16 * MT, false);
  const int o = row * N + n0 + 8 * c;
  const DgIn in = dg_fetch<EPI>(g, o);
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
  dg_finish<EPI>(g, o, n0 + 8 * c, v, v2, in);
}

template <int LAYOUT, int EPI>
hipError_t thin_launch(const DgArgs& a, hipStream_t s) {
  const int M = a.prob[0].M, N = a.prob[0].N;
  const int bn = EPI == kDgGateUp ? 16 : 32;
  const dim3 block(kThinThreads);
#define W4A16_THIN(MT_)                                                                                           \
  hipLaunchKernelGGL((k_gemm_thin<LAYOUT, EPI, MT_>), dim3(8 * (((N + bn - 1) / bn + 7) / 8), (M + 16 * MT_ - 1) / (16 * MT_)), \
                     block, kThinWaves * thin_stages(MT_) * (2048 + 1024 * MT_), s, a)
  if (M <= 16) W4A16_THIN(1);
  else if (M <= 32) W4A16_THIN(2);
  else W4A16_THIN(4);
#undef W4A16_THIN
  return hipGetLastError();
}

}  // namespace w4a16
