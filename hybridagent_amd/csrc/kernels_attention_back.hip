// Gradients of the attention over packed prompts (include/w4a16moe.h,
// w4a16_attention_backward).  With p = exp(scale q k^T - lse) over the seen keys:
//
//   delta = sum over d of dout out      (a query's)
//   dv = p^T dout, ds = p (dout v^T - delta), dq = scale ds k, dk = scale ds^T q
//
// in three launches: delta; dq, with a workgroup's queries in registers and the
// keys and values in tiles; dk and dv, with its keys and values in registers and
// the queries and gradients of all heads of its group in tiles.  The scores are
// computed twice (7 products in place of 5): every sum stays in one workgroup and
// in one order, without atomics.
//
// In the last two a pair of wavefronts of one SIMD shares 16 N rows: the first
// has the scores and p, the second dout v^T and ds.  p, in fp32, and dq's ds pass
// between them through LDS, lane to the same lane.  One wavefront would need the
// rows of both matrices and all sums in its registers: with a quarter of the
// matrix unit's registers for itself, that is half as many rows, and twice the
// LDS reads per product.
#include <type_traits>

#include "attention.hpp"

namespace w4a16 {

namespace {

constexpr int kPairs = 4, kBackThreads = 128 * kPairs;
constexpr int back_slots(int D) { return D == 512 ? 2 : 3; }
// 16-row tiles of a pair
constexpr int dq_rows(int D) { return D == 512 ? 1 : D == 256 ? 2 : 4; }
constexpr int dkv_rows(int D) { return D == 512 ? 1 : D == 256 ? 2 : D == 128 ? 3 : 4; }
template <int D>
constexpr int back_lds(int n) {
  return back_slots(D) * AtFeed<D, 2 * kPairs>::kSlot + kPairs * n * 64 * (2 * 16 + 16);
}

}  // namespace

// delta[h][t]: D / 8 lanes per row
template <typename T, int D>
__global__ __launch_bounds__(256) void k_attention_delta(AttnArgs a) {
  constexpr int L = D / 8;
  const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (row >= (int64_t)a.Tq * a.Hq) return;
  const int64_t at = row * (D * 2) + 16 * (threadIdx.x % L);
  const u32x4_t x = ld16(static_cast<const unsigned char*>(a.dout) + at);
  const u32x4_t y = ld16(static_cast<const unsigned char*>(a.out) + at);
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v = __builtin_fmaf(at_lo<T>(x[i]), at_lo<T>(y[i]), v);
    v = __builtin_fmaf(at_hi<T>(x[i]), at_hi<T>(y[i]), v);
  }
#pragma unroll
  for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o);
  if (threadIdx.x % L == 0) {
    const int64_t t = row / a.Hq;
    a.delta[(row - t * a.Hq) * a.Tq + t] = v;
  }
}

// A workgroup has 16 NQ queries of a head per pair.
template <typename T, int D, int NQ>
__global__ __launch_bounds__(kBackThreads, 2) void k_attention_dq(AttnArgs a) {
  constexpr int kSlots = back_slots(D);
  constexpr int BQ = 16 * NQ * kPairs;
  constexpr int NI = D / 32, ND = D / 32;  // a wavefront sums half of dq's columns
  constexpr int kAhead = 2;
  using Feed = AtFeed<D, 2 * kPairs>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int role = wave / kPairs, place = wave % kPairs;

  const int item = at_swizzle(a.tiles * a.Hq);
  if (item < 0) return;
  const int head = item / a.tiles;
  const AtItem it = at_find(a.cu_q, a.B, a.Tq, BQ, item - head * a.tiles);
  if (it.seq < 0) return;
  int k_first, nk;
  at_rows(a.cu_k, a.B, a.Tk, it.seq, k_first, nk);
  const int nq = it.len, off = nk - nq;
  const int wg0 = (it.tiles - 1 - it.tile) * BQ;
  const int q0 = wg0 + 16 * NQ * place;
  int lo, hi, wlo, whi;
  at_seen_keys(a, nk, off, wg0, min(wg0 + BQ, nq) - 1, lo, hi);
  at_seen_keys(a, nk, off, q0, min(q0 + 16 * NQ, nq) - 1, wlo, whi);
  if (q0 >= nq) whi = 0;
  lo &= ~31;
  const int steps = hi > lo ? (hi - lo + 31) / 32 : 0;

  const unsigned char* kp = static_cast<const unsigned char*>(a.k) + k_first * a.k_stride + (head / a.group) * a.k_head;
  const unsigned char* vp = static_cast<const unsigned char*>(a.v) + k_first * a.v_stride + (head / a.group) * a.v_head;
  Feed feed;
  feed.init(kp, a.k_stride, vp, a.v_stride, wave);
#pragma unroll
  for (int s = 0; s < kSlots - 1; ++s) feed.issue(smem + s * Feed::kSlot, lo + 32 * s, s < steps ? hi : 0, wave);

  // the rows of q (first) or dout; -lse log2(e) or delta
  u32x4_t rows[NQ][NI];
  float stat[NQ];
  f32x4_t acc[ND][NQ];
  const unsigned char* rp = role ? static_cast<const unsigned char*>(a.dout) + head * (D * 2)
                                 : static_cast<const unsigned char*>(a.q) + head * a.q_head;
  const float* sp = (role ? a.delta : a.lse) + (int64_t)head * a.Tq;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int64_t q = it.first + min(q0 + 16 * n + r, nq - 1);
    at_load_row<NI>(rp, q, role ? (int64_t)a.Hq * D * 2 : a.q_stride, rows[n]);
    const float v = sp[q];
    // a query without keys: its scores are all masked
    stat[n] = role ? v : v == -INFINITY ? 0.f : -v * kLog2e;
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  AtLane<D> ln;
  ln.init();
  ln.half_cols(role);
  // the exchange: p [place][tile][n][lane], then ds [place][n][lane]
  f32x4_t* const xp = reinterpret_cast<f32x4_t*>(smem + kSlots * Feed::kSlot) + place * 2 * NQ * 64 + lane;
  u32x4_t* const xd = reinterpret_cast<u32x4_t*>(smem + kSlots * Feed::kSlot) + (kPairs * 2 + place) * NQ * 64 + lane;

  const uint32_t base = at_lds(smem);
  int slot = 0;
  for (int t = 0; t < steps; ++t) {
    __builtin_amdgcn_s_waitcnt(px_vm_wait((kSlots - 2) * Feed::kLoads));
    px_barrier();
    {
      const int ahead = t + kSlots - 1;
      const int to = slot == 0 ? kSlots - 1 : slot - 1;
      feed.issue(smem + to * Feed::kSlot, lo + 32 * ahead, ahead < steps ? hi : 0, wave);
    }
    const uint32_t tile = base + slot * Feed::kSlot;
    slot = slot == kSlots - 1 ? 0 : slot + 1;
    const int key0 = lo + 32 * t;
    const bool active = key0 < whi && key0 + 32 > wlo;
    f32x4_t s[2][NQ];
    if (active) {
      at_scores<T, kAhead>(ln, tile + (role ? at_tile_bytes<D>() : 0), rows, s);
      if (!role) {
        if (key0 + 32 > nk || (a.causal && key0 + 31 > q0 + off) ||
            (a.window > 0 && key0 <= min(q0 + 16 * NQ, nq) - 1 + off - a.window)) {
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            const int q = q0 + 16 * n + r + off;
            const int last = a.causal ? min(nk - 1, q) : nk - 1;
            const int first = a.window > 0 ? q - a.window + 1 : 0;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int key = key0 + 8 * c + 4 * u + i;
                s[u][n][i] = key <= last && key >= first ? s[u][n][i] : -INFINITY;
              }
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              s[u][n][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][n][i], a.scale2, stat[n]));
            xp[(u * NQ + n) * 64] = s[u][n];
          }
      }
    }
    px_barrier();
    u32x4_t p[NQ];
    if (active && role) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const f32x4_t w = xp[(u * NQ + n) * 64];
          // (a masked key's dout v^T may be anything)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[u][n][i] = w[i] == 0.f ? 0.f : w[i] * (s[u][n][i] - stat[n]);
        }
        p[n] = at_pack8<T>(s[0][n], s[1][n]);
        xd[n * 64] = p[n];
      }
    }
    px_barrier();
    if (active) {
      if (!role) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) p[n] = xd[n * 64];
      }
      at_accumulate<T, kAhead>(ln, tile, p, acc);
    }
  }

#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int q = q0 + 16 * n + r;
    if (q >= nq) continue;
    unsigned char* o =
        static_cast<unsigned char*>(a.dq) + ((int64_t)(it.first + q) * a.Hq + head) * (D * 2) + role * D + 8 * c;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const f32x4_t v = acc[d][n] * a.scale;
      *reinterpret_cast<u32x2_t*>(o + 32 * d) = u32x2_t{at_pack2<T>(v[0], v[1]), at_pack2<T>(v[2], v[3])};
    }
  }
}

// A workgroup has 16 NK keys of a key-value head per pair; the first wavefront
// sums dv, the second dk.
template <typename T, int D, int NK>
__global__ __launch_bounds__(kBackThreads, 2) void k_attention_dkv(AttnArgs a) {
  constexpr int kSlots = back_slots(D);
  constexpr int BK = 16 * NK * kPairs;
  constexpr int NI = D / 32, ND = D / 16;
  constexpr int kAhead = 2;
  using Feed = AtFeed<D, 2 * kPairs>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int role = wave / kPairs, place = wave % kPairs;

  const int item = at_swizzle(a.tiles * a.Hk);
  if (item < 0) return;
  const int kvh = item / a.tiles;
  const AtItem it = at_find(a.cu_k, a.B, a.Tk, BK, item - kvh * a.tiles);
  if (it.seq < 0) return;
  int q_first, nq;
  at_rows(a.cu_q, a.B, a.Tq, it.seq, q_first, nq);
  const int nk = it.len, off = nk - nq;
  const int wg0 = it.tile * BK;  // the first keys are seen by the most queries
  const int k0 = wg0 + 16 * NK * place;
  // the queries lo .. hi - 1 that see a range of keys
  auto range = [&](int first, int last, int& lo, int& hi) {
    lo = a.causal ? max(0, first - off) : 0;
    hi = a.window > 0 ? min(nq, last - off + a.window) : nq;
  };
  int lo, hi, wlo, whi;
  range(wg0, min(wg0 + BK, nk) - 1, lo, hi);
  range(k0, min(k0 + 16 * NK, nk) - 1, wlo, whi);
  if (k0 >= nk) whi = 0;
  lo &= ~31;
  const int per = hi > lo ? (hi - lo + 31) / 32 : 0;  // steps of a head
  const int steps = per * a.group;

  struct Next {
    int head, q0;
  } next{kvh * a.group, lo};
  const int64_t g_stride = (int64_t)a.Hq * D * 2;
  const unsigned char* qp = static_cast<const unsigned char*>(a.q) + q_first * a.q_stride;
  const unsigned char* gp = static_cast<const unsigned char*>(a.dout) + q_first * g_stride;
  Feed feed;
  feed.init(qp, a.q_stride, gp, g_stride, wave);
  // the next step's loads, of a head after the other
  auto issue = [&](unsigned char* to, bool any) {
    feed.issue(to, next.q0, any ? nq : 0, wave, next.head * a.q_head, next.head * (D * 2));
    next.q0 += 32;
    if (next.q0 >= hi) {
      next.q0 = lo;
      ++next.head;
    }
  };
#pragma unroll
  for (int s = 0; s < kSlots - 1; ++s) issue(smem + s * Feed::kSlot, s < steps);

  u32x4_t rows[NK][NI];  // of k (first) or v
  f32x4_t acc[ND][NK];
  const unsigned char* rp = role ? static_cast<const unsigned char*>(a.v) + kvh * a.v_head
                                 : static_cast<const unsigned char*>(a.k) + kvh * a.k_head;
#pragma unroll
  for (int n = 0; n < NK; ++n) {
    at_load_row<NI>(rp, it.first + min(k0 + 16 * n + r, nk - 1), role ? a.v_stride : a.k_stride, rows[n]);
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  AtLane<D> ln;
  ln.init();
  f32x4_t* const xp = reinterpret_cast<f32x4_t*>(smem + kSlots * Feed::kSlot) + place * 2 * NK * 64 + lane;

  // lse or delta of a lane's eight queries; past the last query zeros
  struct Stats {
    u32x4_t v[2];
  };
  const float* sp = (role ? a.delta : a.lse) + q_first;
  auto fetch = [&](int head, int q0) {
    Stats st;
    const auto x = make_rsrc(sp + (int64_t)head * a.Tq + q0, (uint32_t)max(nq - q0, 0) * 4u);
#pragma unroll
    for (int u = 0; u < 2; ++u) st.v[u] = buf_ld16(x, 32 * c, 16 * u);
    return st;
  };
  int head = kvh * a.group, q0 = lo;
  Stats now = fetch(head, steps > 0 ? q0 : nq);

  const uint32_t base = at_lds(smem);
  int slot = 0;
  for (int t = 0; t < steps; ++t) {
    __builtin_amdgcn_s_waitcnt(px_vm_wait((kSlots - 2) * Feed::kLoads));
    px_barrier();
    const int at = q0;
    q0 += 32;
    if (q0 >= hi) {
      q0 = lo;
      ++head;
    }
    issue(smem + (slot == 0 ? kSlots - 1 : slot - 1) * Feed::kSlot, t + kSlots - 1 < steps);
    const uint32_t tile = base + slot * Feed::kSlot;
    slot = slot == kSlots - 1 ? 0 : slot + 1;
    const bool active = at < whi && at + 32 > wlo;
    f32x4_t s[2][NK];
    if (active) {
      at_scores<T, kAhead>(ln, tile + (role ? at_tile_bytes<D>() : 0), rows, s);
      if (!role) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float lse2 = __uint_as_float(now.v[u][i]) * kLog2e;
#pragma unroll
            for (int n = 0; n < NK; ++n)
              s[u][n][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][n][i], a.scale2, -lse2));
          }
        if (at + 32 > nq || k0 + 16 * NK > nk || (a.causal && k0 + 16 * NK - 1 > at + off) ||
            (a.window > 0 && k0 <= at + 31 + off - a.window)) {
#pragma unroll
          for (int n = 0; n < NK; ++n) {
            // the queries low .. high of the step see the key
            const int key = k0 + 16 * n + r;
            const int low = a.causal ? key - off - at : 0;
            const int high = key >= nk ? -1 : (a.window > 0 ? min(nq, key - off + a.window) : nq) - 1 - at;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int q = 8 * c + 4 * u + i;
                s[u][n][i] = q >= low && q <= high ? s[u][n][i] : 0.f;
              }
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int n = 0; n < NK; ++n) xp[(u * NK + n) * 64] = s[u][n];
      }
    }
    px_barrier();
    if (active && role) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int n = 0; n < NK; ++n) {
          const f32x4_t w = xp[(u * NK + n) * 64];
          // (a masked query's dout v^T may be anything)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[u][n][i] = w[i] == 0.f ? 0.f : w[i] * (s[u][n][i] - __uint_as_float(now.v[u][i]));
        }
    }
    now = fetch(t + 1 < steps ? head : kvh * a.group, t + 1 < steps ? q0 : nq);
    if (!active) continue;
    u32x4_t p[NK];
#pragma unroll
    for (int n = 0; n < NK; ++n) p[n] = at_pack8<T>(s[0][n], s[1][n]);
    at_accumulate<T, kAhead>(ln, tile + (role ? 0 : at_tile_bytes<D>()), p, acc);
  }

  unsigned char* const out = static_cast<unsigned char*>(role ? a.dk : a.dv);
  const float scale = role ? a.scale : 1.f;
#pragma unroll
  for (int n = 0; n < NK; ++n) {
    const int k = k0 + 16 * n + r;
    if (k >= nk) continue;
    unsigned char* o = out + ((int64_t)(it.first + k) * a.Hk + kvh) * (D * 2) + 8 * c;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const f32x4_t v = acc[d][n] * scale;
      *reinterpret_cast<u32x2_t*>(o + 32 * d) = u32x2_t{at_pack2<T>(v[0], v[1]), at_pack2<T>(v[2], v[3])};
    }
  }
}

namespace {

template <typename T, int D>
hipError_t back(AttnArgs a, hipStream_t s) {
  constexpr int NQ = dq_rows(D), NK = dkv_rows(D);
  static_assert(back_lds<D>(NQ) <= 160 * 1024 && back_lds<D>(NK) <= 160 * 1024, "a CU's LDS");
  if (a.Tq > 0) {
    const int64_t rows = (int64_t)a.Tq * a.Hq, per = 256 / (D / 8);
    hipLaunchKernelGGL((k_attention_delta<T, D>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, s, a);
  }
  if (a.Tq > 0 && a.dq != nullptr) {
    a.tiles = a.Tq / (16 * NQ * kPairs) + a.B + 1;
    hipLaunchKernelGGL((k_attention_dq<T, D, NQ>), dim3(at_grid((int64_t)a.tiles * a.Hq)), dim3(kBackThreads),
                       back_lds<D>(NQ), s, a);
  }
  if (a.Tk > 0 && a.dk != nullptr) {
    a.tiles = a.Tk / (16 * NK * kPairs) + a.B + 1;
    hipLaunchKernelGGL((k_attention_dkv<T, D, NK>), dim3(at_grid((int64_t)a.tiles * a.Hk)), dim3(kBackThreads),
                       back_lds<D>(NK), s, a);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t back_type(const AttnArgs& a, hipStream_t s) {
  switch (a.D) {
    case 64: return back<T, 64>(a, s);
    case 128: return back<T, 128>(a, s);
    case 256: return back<T, 256>(a, s);
    case 512: return back<T, 512>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_attention_backward(int dtype, const AttnArgs& a, hipStream_t s) {
  return dtype == 0 ? back_type<__bf16>(a, s) : back_type<_Float16>(a, s);
}

}  // namespace w4a16
