// Attention over packed prompts: out = softmax(scale q k^T) v over the keys that
// a query sees, with grouped heads, sequences of any lengths packed one behind
// the other, causal masks and windows (include/w4a16moe.h, w4a16_attention).
#include <type_traits>

#include "attention.hpp"

namespace w4a16 {

namespace {

// Two groups of four wavefronts, one of each on every SIMD, take turns: while one
// is at the matrix units (X: the last step's weights times values, then this
// step's scores), the other turns scores into weights (Y), a barrier between the
// phases.  Group B runs a phase behind A:
//
//   phase      2t             2t + 1         2t + 2
//   A          X(t)           Y(t)           X(t + 1)
//   B          Y(t - 1)       X(t)           Y(t)
//
// so keys t are read in the phases 2t and 2t + 1, values t in 2t + 2 and 2t + 3.
// A loads the keys and B the values, each at the start of an even phase: into the
// ring's slot that the step S before left, for S - 1 steps ahead.
constexpr int kGroup = 4, kWaves = 2 * kGroup;

template <int D>
constexpr int fwd_slots() { return D == 512 ? 2 : 3; }

}  // namespace

// A workgroup has 16 NQ queries of a head per wavefront; PAIR: per pair of
// wavefronts of a group, each with half of D: of the scores' sum, whose halves
// they exchange through LDS between the phases, and of the output's columns.
// (Heads of 512: a wavefront's registers hold 16 queries' output and the queries,
// and every operand read from LDS would feed one matrix instruction.)
template <typename T, int D, int NQ, bool PAIR>
__global__ __launch_bounds__(64 * kWaves, 2) void k_attention(AttnArgs a) {
  constexpr int S = fwd_slots<D>();
  constexpr int kHalves = PAIR ? 2 : 1;
  constexpr int BQ = 16 * NQ * kWaves / kHalves;
  constexpr int NI = D / 32 / kHalves, ND = D / 16 / kHalves;
  constexpr int kTile = at_tile_bytes<D>();
  constexpr int kAhead = 4;
  using Feed = AtFeed<D, kGroup>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool second = wave >= kGroup;  // group B
  const int half = PAIR ? wave & 1 : 0;

  const AtPlace at = at_place(a.Hq);
  const AtItem it = at_find(a.cu_q, a.B, a.Tq, BQ, at.rank);
  if (it.seq < 0) return;
  int k_first, nk;
  at_rows(a.cu_k, a.B, a.Tk, it.seq, k_first, nk);
  const int nq = it.len, off = nk - nq;
  const int wg0 = it.level * BQ;
  const int q0 = wg0 + 16 * NQ * (wave / kHalves);

  int lo, hi, wlo, whi;
  at_seen_keys(a, nk, off, wg0, min(wg0 + BQ, nq) - 1, lo, hi);
  at_seen_keys(a, nk, off, q0, min(q0 + 16 * NQ, nq) - 1, wlo, whi);
  if (q0 >= nq) whi = 0;
  lo &= ~31;
  const int steps = hi > lo ? (hi - lo + 31) / 32 : 0;

  // its keys (A) or values (B), and their ring
  Feed feed;
  {
    const int kvh = at.head / a.group;
    if (second)
      feed.init(static_cast<const unsigned char*>(a.v) + k_first * a.v_stride + kvh * a.v_head, a.v_stride,
                wave - kGroup);
    else
      feed.init(static_cast<const unsigned char*>(a.k) + k_first * a.k_stride + kvh * a.k_head, a.k_stride, wave);
  }
  unsigned char* const ring = smem + (second ? S * kTile : 0);
#pragma unroll
  for (int s = 0; s < S - 1; ++s) feed.issue(ring + s * kTile, lo + 32 * s, s < steps ? hi : 0);

  u32x4_t qf[NQ][NI];
  float m[NQ], l[NQ];
  f32x4_t acc[ND][NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    at_load_row<NI>(static_cast<const unsigned char*>(a.q) + at.head * a.q_head + half * D,
                    it.first + min(q0 + 16 * n + r, nq - 1), a.q_stride, qf[n]);
    m[n] = -1e30f;  // below every score's, so that a masked key's weight is zero
    l[n] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  AtLane<D> ln;
  ln.init();
  if constexpr (PAIR) {
    ln.half_rows(half);
    ln.half_cols(half);
  }
  // the pairs' exchange: [wave][tile][n][lane]
  f32x4_t* const mine = reinterpret_cast<f32x4_t*>(smem + 2 * S * kTile) + wave * 2 * NQ * 64 + lane;
  const f32x4_t* const other = mine + (half ? -1 : 1) * 2 * NQ * 64;
  const uint32_t base = at_lds(smem);

  f32x4_t s[2][NQ];
  u32x4_t p[NQ];
  bool active = false;  // the last step had keys that the wavefront's queries see
  if (second) px_barrier();
  int slot = 0, last = S - 1;  // of step t, of the step before (and of the next to load)
  for (int t = 0; t < steps; ++t) {
    if (!second) __builtin_amdgcn_s_waitcnt(px_vm_wait((S - 2) * Feed::kLoads));
    px_barrier();
    const int ahead = t + S - 1;
    if (!second) feed.issue(ring + last * kTile, lo + 32 * ahead, ahead < steps ? hi : 0);
    if (active) at_accumulate<T, kAhead>(ln, base + (S + last) * kTile, p, acc);
    const int key0 = lo + 32 * t;
    active = key0 < whi && key0 + 32 > wlo;
    if (active) {
      at_scores<T, kAhead>(ln, base + slot * kTile, qf, s);
      if constexpr (PAIR) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int n = 0; n < NQ; ++n) mine[(u * NQ + n) * 64] = s[u][n];
      }
    }
    if (second) __builtin_amdgcn_s_waitcnt(px_vm_wait((S - 2) * Feed::kLoads));
    px_barrier();
    if (second) feed.issue(ring + last * kTile, lo + 32 * ahead, ahead < steps ? hi : 0);
    last = slot;
    slot = slot == S - 1 ? 0 : slot + 1;
    if (!active) continue;
    if constexpr (PAIR) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[u][n] += other[(u * NQ + n) * 64];
    }
    // some query does not see some key
    if (key0 + 32 > nk || (a.causal && key0 + 31 > q0 + off) ||
        (a.window > 0 && key0 <= min(q0 + 16 * NQ, nq) - 1 + off - a.window)) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int q = q0 + 16 * n + r + off;
        const int to = a.causal ? min(nk - 1, q) : nk - 1;
        const int from = a.window > 0 ? q - a.window + 1 : 0;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = key0 + 8 * c + 4 * u + i;
            s[u][n][i] = key <= to && key >= from ? s[u][n][i] : -INFINITY;
          }
      }
    }
    // the running maximum moves where a score is 2^8 above it: the weights stay
    // below 2^8 of the sum's first
    float top[NQ];
    bool over = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      top[n] = fmaxf(fmaxf(fmaxf(s[0][n][0], s[0][n][1]), fmaxf(s[0][n][2], s[0][n][3])),
                     fmaxf(fmaxf(s[1][n][0], s[1][n][1]), fmaxf(s[1][n][2], s[1][n][3]))) *
               a.scale2;
      over |= top[n] > m[n] + 8.f;
    }
    if (__any(over)) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const float now = fmaxf(m[n], at_max_over_c(top[n]));
        const float f = __builtin_amdgcn_exp2f(m[n] - now);
        m[n] = now;
        l[n] *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d][n] *= f;
      }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[u][n][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][n][i], a.scale2, -m[n]));
          l[n] += s[u][n][i];
        }
      p[n] = at_pack8<T>(s[0][n], s[1][n]);
    }
  }
  if (!second) px_barrier();
  if (active) at_accumulate<T, kAhead>(ln, base + (S + last) * kTile, p, acc);

#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int q = q0 + 16 * n + r;
    const float sum = at_sum_over_c(l[n]);
    if (q >= nq) continue;
    const float f = sum == 0.f ? 0.f : 1.0f / sum;
    if (a.lse != nullptr && c == 0 && half == 0)
      a.lse[(int64_t)at.head * a.Tq + it.first + q] = (m[n] + __builtin_amdgcn_logf(sum)) * kLn2;
    unsigned char* o =
        static_cast<unsigned char*>(a.out) + ((int64_t)(it.first + q) * a.Hq + at.head) * (D * 2) + half * D + 8 * c;
#pragma unroll
    for (int d = 0; d < ND; ++d)
      *reinterpret_cast<u32x2_t*>(o + 32 * d) =
          u32x2_t{at_pack2<T>(acc[d][n][0] * f, acc[d][n][1] * f), at_pack2<T>(acc[d][n][2] * f, acc[d][n][3] * f)};
  }
}

namespace {

template <typename T, int D, int NQ, bool PAIR>
hipError_t fwd(AttnArgs a, hipStream_t s) {
  a.tiles = a.Tq / (16 * NQ * kWaves / (PAIR ? 2 : 1)) + a.B + 1;
  constexpr int lds = 2 * fwd_slots<D>() * at_tile_bytes<D>() + (PAIR ? kWaves * 2 * NQ * 64 * 16 : 0);
  static_assert(lds <= 160 * 1024, "a CU's LDS");
  hipLaunchKernelGGL((k_attention<T, D, NQ, PAIR>), dim3((unsigned)(a.tiles * a.Hq)), dim3(64 * kWaves), lds, s, a);
  return hipGetLastError();
}

template <typename T>
hipError_t fwd_type(const AttnArgs& a, hipStream_t s) {
  switch (a.D) {
    case 64: return fwd<T, 64, 2, false>(a, s);
    case 128: return fwd<T, 128, 2, false>(a, s);
    case 256: return fwd<T, 256, 2, false>(a, s);
    case 512: return fwd<T, 512, 2, true>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_attention(int dtype, const AttnArgs& a, hipStream_t s) {
  return dtype == 0 ? fwd_type<__bf16>(a, s) : fwd_type<_Float16>(a, s);
}

}  // namespace w4a16
