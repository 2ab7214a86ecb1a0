// Gradients of the attention over packed prompts (include/w4a16moe.h,
// w4a16_attention_backward).  With p = exp(scale q k^T - lse) over the seen keys:
//
//   delta = sum over d of dout out      (a query's; of out as it was rounded: the forward
//                                        pass keeps no other)
//   dv = p^T dout, ds = p (dout v^T - delta), dq = scale ds k, dk = scale ds^T q
//
// in two launches: delta and dq, with a workgroup's queries in registers and the
// keys and values in tiles; dk and dv, with its keys and values in registers and
// the queries and gradients of all heads of its group in tiles.  The scores are
// computed twice (7 products in place of 5): every sum stays in one workgroup, or in
// the few that share a tile's steps (attn_split) and a join of theirs, and in one
// order, without atomics.
//
// In the last two a pair of wavefronts of one SIMD shares 16 N rows: A has the
// scores and p, B dout v^T and ds.  p, in fp32, and dq's ds pass between them
// through LDS, lane to the same lane.  (One wavefront would need the rows of both
// matrices and all sums in its registers: with its half of the SIMD's that is half
// as many rows, and twice the LDS reads per product.)  They take turns at the
// matrix units, a barrier between the phases: X is the sums of a step before and
// this step's scores (or dout v^T), Y turns these into p (or ds).
//
//   phase    2t           2t + 1       2t + 2
//   A        X(t)         Y(t): p(t)   X(t + 1)
//   B        Y(t - 1)     X(t)         Y(t): ds(t) from p(t)
//
// A step's tiles are in LDS until the last of their reads, three phases on (dk:
// queries in X(t + 1) of B), four (dq: keys in X(t + 2) of A, which has ds from B)
// or one.  Heads of 512 have no room for as many: there both have their scores,
// then p, ds and the sums of one step, a barrier between.
//
// Bound: the phases.  Of heads of 256 dq's X takes 1500 cycles for 768 of matrix
// instructions, dkv's as forward; of 64 and 128 Y, the exponentials and the exchange,
// is the longer (matrix units busy 0.32 and 0.39 of the CUs' cycles in dq, 0.29 and 0.43 in
// dkv).  2 x 4096 tokens, 16 heads, 8 key-value heads, TFLOP/s of the three products
// of dq, and of the four of dk and dv: heads of 64 148 us (696) and 260 (528), 128 240
// (859) and 395 (696), 256 383-396 (1060) and 475-490 (1140), 512 925-960 (875) and
// 1130-1183 (950).  Of the five that the gradients cannot do without: 430, 550, 790 and
// 660.  fp16 with its powers (below): 176 and 283, 261 and 411, 408 and 512, 970 and 1215.
#include <type_traits>

#include "attention.hpp"

namespace w4a16 {

namespace {

constexpr int kPairs = 4, kBackThreads = 128 * kPairs;
constexpr bool phases(int D) { return D < 512; }
// 16-row tiles of a pair
constexpr int back_rows(int D, bool low) { return attn_rows(kAttnDq, D, low) / (16 * kPairs); }
// LDS slots of A's tiles (keys, queries) and of B's (values, dout)
constexpr int slots_a(int D) { return phases(D) ? 4 : 2; }
constexpr int slots_b(int D) { return phases(D) ? 3 : 2; }
// and bytes, with the exchange
constexpr int back_lds(int D, int n) {
  return (slots_a(D) + slots_b(D)) * 64 * D + kPairs * n * 64 * (2 * 16 + 16 + 4);
}

__device__ __forceinline__ int ring_next(int slot, int slots) { return slot == slots - 1 ? 0 : slot + 1; }

}  // namespace

// ds as an operand.  fp16 has numbers of 2^-24 .. 2^16 and ds follows dout's size, whatever that
// is: rounded as it is, with dout of 3e-5 over 1500 keys elements of dq and dk were off by up to
// 300 times their rounding, and above 65504 infinite.  So a column's ds carry a power of two, as a
// softmax its maximum: the largest so far makes 2^7 or more of it, and when one exceeds 2^15 the
// column's sums take a lower power.  What is then below fp16's numbers is 2^-32 of the largest.
// (bf16 has fp32's range.)  The first power leaves fp32 room for any ds of fp16 numbers.
template <typename T>
constexpr bool kLift = std::is_same_v<T, _Float16>;
constexpr float kFirstLift = 0x1p64f;
// p as the operand of dv in fp16 lies 2^12 higher: 1 / n of n equal weights is below fp16's normal
// numbers from 16385 on (818400 of them: dv off by 2.5 %), with 2^12 of no number of keys.  Not
// higher: of scores of 10^7 fp32's roundings leave a p of one up to a few times as large, which must
// stay below 65504.  ds, made of it, has the 2^12 too.
template <typename T>
constexpr float kWeightLift = kLift<T> ? 12.f : 0.f;
// the power of two that takes `top` to 2^7 .. 2^8
__device__ __forceinline__ float lift_for(float top) {
  return __uint_as_float((uint32_t)(261 - max((int)(__float_as_uint(top) >> 23), 8)) << 23);
}
// Columns N0 .. N1 - 1 of ds at their powers: where one exceeds the bound all take lower
// ones, the sums too.  True: powers changed.
template <int N0, int N1, int ND, int N>
__device__ __forceinline__ bool fit_slopes(f32x4_t (&s)[2][N], f32x4_t (&acc)[ND][N], float (&lift)[N]) {
  float top[N];
  bool over = false;
#pragma unroll
  for (int n = N0; n < N1; ++n) {
    top[n] = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) top[n] = fmaxf(top[n], fabsf(s[u][n][i]));
    over |= top[n] > 0x1p15f;
  }
  if (!__any(over)) return false;
#pragma unroll
  for (int n = N0; n < N1; ++n) {
    const float t = at_max_over_c(top[n]), f = t > 0x1p15f ? lift_for(t) : 1.f;
    lift[n] *= f;
    s[0][n] *= f;
    s[1][n] *= f;
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d][n] *= f;
  }
  return true;
}
// the sums as they are, of sums with a power
template <typename T, int ND, int N>
__device__ __forceinline__ void unlift(f32x4_t (&acc)[ND][N], const float (&lift)[N], float more = 1.f) {
  if constexpr (kLift<T>)
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const float f = more / lift[n];
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d][n] *= f;
    }
}

// delta of row r, in lane c's chunks of dout's row and out's
template <typename T, int NI>
__device__ __forceinline__ float row_delta(const u32x4_t (&x)[NI], const u32x4_t (&y)[NI]) {
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      v = __builtin_fmaf(at_lo<T>(x[i][w]), at_lo<T>(y[i][w]), v);
      v = __builtin_fmaf(at_hi<T>(x[i][w]), at_hi<T>(y[i][w]), v);
    }
  return at_sum_over_c(v);
}

// delta[h][t], where dq is not wanted: a wavefront has 16 rows
template <typename T, int D>
__global__ __launch_bounds__(256) void k_attention_delta(AttnArgs a) {
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int64_t rows = (int64_t)a.Tq * a.Hq, row = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16 + r;
  u32x4_t x[D / 32], y[D / 32];
  at_load_row<D / 32>(static_cast<const unsigned char*>(a.dout), min(row, rows - 1), D * 2, x);
  at_load_row<D / 32>(static_cast<const unsigned char*>(a.out), min(row, rows - 1), D * 2, y);
  const float v = row_delta<T>(x, y);
  if (c == 0 && row < rows) {
    const int64_t t = row / a.Hq;
    a.delta[(row - t * a.Hq) * a.Tq + t] = v;
  }
}

// A lane's columns of a row's gradient: the output's `ok` row at `at`, or a part's of
// it, which lie `plane` floats apart.
template <typename T, int ND, int N>
__device__ __forceinline__ void back_store(const f32x4_t (&acc)[ND][N], int n, bool ok, void* out, float* parts,
                                           int64_t plane, const AtPart& part, int64_t at, int c, float scale) {
  if (part.of == 1) {
    unsigned char* o = static_cast<unsigned char*>(out) + 2 * (at + at_pair_column(c));
#pragma unroll
    for (int d = 0; d < ND; d += 2) {
      const u32x4_t v = at_pair<T>(acc[d][n] * scale, acc[d + 1][n] * scale);
      if (ok) *reinterpret_cast<u32x4_t*>(o + 32 * d) = v;
    }
  } else if (ok) {
    float* o = parts + part.index * plane + at + 4 * c;
#pragma unroll
    for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4_t*>(o + 16 * d) = acc[d][n];
  }
}

// join_rows rows of a sequence, from `row` on, joined (several rows a thread, as in the
// forward pass, are slower here: more parts, fewer tiles)
constexpr int join_rows(int D) { return 1024 / D; }
template <typename T, int D>
__device__ __forceinline__ void back_join(const float* parts, int64_t plane, int n, int first, int row, int len,
                                          int heads, int head, float scale, void* out) {
  constexpr int L = D / 4;
  const int i = row + threadIdx.x / L;
  if (i >= len) return;
  const int64_t at = ((int64_t)(first + i) * heads + head) * D + 4 * (threadIdx.x % L);
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int p = 0; p < n; ++p) v += *reinterpret_cast<const f32x4_t*>(parts + p * plane + at);
  v *= scale;
  *reinterpret_cast<u32x2_t*>(static_cast<unsigned char*>(out) + 2 * at) =
      u32x2_t{at_pack2<T>(v[0], v[1]), at_pack2<T>(v[2], v[3])};
}

// A workgroup has 16 NQ queries of a head per pair.
template <typename T, int D, int NQ>
__global__ __launch_bounds__(kBackThreads, 2) void k_attention_dq(AttnArgs a) {
  constexpr int SA = slots_a(D), SB = slots_b(D), S = SA + SB;
  constexpr int BQ = 16 * NQ * kPairs;
  constexpr int NI = D / 32, ND = D / 32;  // a wavefront sums half of dq's columns
  constexpr int kTile = at_tile_bytes<D>();
  constexpr int kAhead = D == 256 ? 4 : 2;  // (2: 384 us where 4 take 375; dk and dv have no room)
  // steps that the loads are ahead, in the second phase (B's in its first: 334 us of
  // heads of 256 in place of 311)
  constexpr int kAheadA = phases(D) ? SA - 2 : 1, kAheadB = SB - 1;
  using Feed = AtFeed<D, kPairs>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int role = wave / kPairs, place = wave % kPairs;

  const AtPlace wg = at_place(a.Hq);
  const int head = wg.head;
  const int index = __builtin_amdgcn_readfirstlane(wg.rank / a.tiles), tile = wg.rank - index * a.tiles;
  const AtItem it = at_find(a.cu_q, a.B, a.Tq, BQ, tile);
  if (it.seq < 0) return;
  int k_first, nk;
  at_rows(a.cu_k, a.B, a.Tk, it.seq, k_first, nk);
  const int nq = it.len, off = nk - nq;
  const int wg0 = it.level * BQ;
  const int q0 = wg0 + 16 * NQ * place;
  int wlo, whi;
  at_seen_keys(a, nk, off, q0, min(q0 + 16 * NQ, nq) - 1, wlo, whi);
  if (q0 >= nq) whi = 0;
  const AtSpan span = at_key_span(a, nk, off, wg0, BQ, nq, 32);
  const AtPart part = at_part(a, span.steps, index);
  if (part.index >= part.of) return;
  const int lo = span.lo + 32 * part.first, hi = span.hi, steps = part.steps;

  Feed feed;
  {
    const int kvh = head / a.group;
    if (role)
      feed.init(static_cast<const unsigned char*>(a.v) + k_first * a.v_stride + kvh * a.v_head, a.v_stride, place);
    else
      feed.init(static_cast<const unsigned char*>(a.k) + k_first * a.k_stride + kvh * a.k_head, a.k_stride, place);
  }
  feed.seek(lo, hi);
  unsigned char* const ring = smem + (role ? SA * kTile : 0);
  int load = 0, to = 0;  // the next step to load, its slot
  auto issue = [&] {
    feed.issue(ring + to * kTile, load < steps);
    feed.skip(1);
    ++load;
    to = ring_next(to, role ? SB : SA);
  };
#pragma unroll
  for (int s = 0; s < (kAheadA > kAheadB ? kAheadA : kAheadB); ++s)
    if (s < (role ? kAheadB : kAheadA)) issue();

  // the rows of q (A) or dout; -lse log2(e) or delta
  u32x4_t rows[NQ][NI];
  float stat[NQ];
  f32x4_t acc[ND][NQ];
  {
    const unsigned char* rp = role ? static_cast<const unsigned char*>(a.dout) + head * (D * 2)
                                   : static_cast<const unsigned char*>(a.q) + head * a.q_head;
    const float* lse = a.lse + (int64_t)head * a.Tq;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int64_t q = it.first + min(q0 + 16 * n + r, nq - 1);
      at_load_row<NI>(rp, q, role ? (int64_t)a.Hq * D * 2 : a.q_stride, rows[n]);
      if (role) {
        u32x4_t out[NI];
        at_load_row<NI>(static_cast<const unsigned char*>(a.out) + head * (D * 2), q, (int64_t)a.Hq * D * 2, out);
        stat[n] = row_delta<T>(rows[n], out);
        if (part.index == 0 && c == 0 && q0 + 16 * n + r < nq) a.delta[(int64_t)head * a.Tq + q] = stat[n];
      } else {
        // a query without keys: its scores are all masked (one whose scores are all -infinity
        // has p not a number here, as in dk and dv)
        stat[n] = lse[q] == -INFINITY && !at_sees(a, nk, off, (int)q - it.first) ? 0.f : -lse[q] * kLog2e;
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
  at_settle(rows);
  at_settle(stat);
  AtLane<D> ln;
  ln.init();
  ln.half_cols(role);
  // the exchange: p [place][tile][n][lane], then ds [place][n][lane] and (fp16) its powers
  f32x4_t* const xp = reinterpret_cast<f32x4_t*>(smem + S * kTile) + place * 2 * NQ * 64 + lane;
  u32x4_t* const xd = reinterpret_cast<u32x4_t*>(smem + S * kTile) + (kPairs * 2 + place) * NQ * 64 + lane;
  float* const xl = reinterpret_cast<float*>(smem + S * kTile + kPairs * 3 * NQ * 64 * 16) + place * NQ * 64 + lane;
  float lift[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    lift[n] = kFirstLift;
    if (kLift<T> && role) {
      stat[n] *= kFirstLift;
      xl[n * 64] = kFirstLift;
    }
  }
  const uint32_t base = at_lds(smem);
  f32x4_t s[2][NQ];
  u32x4_t p[NQ];

  auto active_at = [&](int t) { return lo + 32 * t < whi && lo + 32 * t + 32 > wlo; };
  // X: ds times the keys in slot `from`, and the scores, or dout v^T, of the step
  // whose tiles are in ka, vb
  auto products = [&](auto role, bool sum, bool scores, int from, int ka, int vb) {
    const uint32_t v = base + from * kTile, w = base + (role ? SA + vb : ka) * kTile;
    u32x4_t next[kAhead];
    if (sum)
      at_accumulate<T, NI>(ln, v, p, acc, w, next);
    else
      at_scores_first<NI>(ln, w, next);
    if (scores) at_scores<T>(ln, w, rows, s, next);
  };
  auto weights = [&](int t) {  // A
    const int key0 = lo + 32 * t;
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
  };
  auto slopes = [&] {  // B
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const f32x4_t w = xp[(u * NQ + n) * 64];
        // (a masked key's weight is zero, and its row one of the sequence's own; delta
        // has the column's power already)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[u][n][i] = w[i] * (kLift<T> ? __builtin_fmaf(s[u][n][i], lift[n], -stat[n]) : s[u][n][i] - stat[n]);
      }
    if constexpr (kLift<T>) {
      float last[NQ];
#pragma unroll
      for (int n = 0; n < NQ; ++n) last[n] = lift[n];
      if (fit_slopes<0, NQ>(s, acc, lift)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          stat[n] *= lift[n] / last[n];
          xl[n * 64] = lift[n];
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      p[n] = at_pack8<T>(s[0][n], s[1][n]);
      xd[n * 64] = p[n];
    }
  };
  auto take = [&] {  // A: ds from B
    if constexpr (kLift<T>) {
      float now[NQ];
      bool other = false;
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        now[n] = xl[n * 64];
        other |= now[n] != lift[n];
      }
      if (__any(other)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const float f = now[n] / lift[n];
          lift[n] = now[n];
#pragma unroll
          for (int d = 0; d < ND; ++d) acc[d][n] *= f;
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) p[n] = xd[n * 64];
  };

  // (each role's loop by itself: in one the compiler copies registers where they meet)
  auto run = [&](auto role) {
    if constexpr (phases(D)) {
      // slots of the keys of step t and of the two before
      int ka = 0, ka1 = SA - 1, ka2 = SA - 2, vb = 0;
      bool now = false, before = false;  // whether the steps t - 1, t - 2 were active
      if (role) px_barrier();
      for (int t = 0; t < steps; ++t) {
        static_assert(kAheadA == kAheadB, "one wait for both");
        __builtin_amdgcn_s_waitcnt(px_vm_wait((kAheadA - 1) * Feed::kLoads));
        px_barrier();
        const bool sum = role ? now : before;
        before = now;
        now = active_at(t);
        __builtin_amdgcn_s_setprio(1);
        products(role, sum, now, role ? ka1 : ka2, ka, vb);
        __builtin_amdgcn_s_setprio(0);
        px_barrier();
        issue();
        if (!role) {
          if (now) weights(t);
          if (before) take();
        } else if (now) {
          slopes();
        }
        ka2 = ka1;
        ka1 = ka;
        ka = ring_next(ka, SA);
        vb = ring_next(vb, SB);
      }
      // ka1: the last step's
      px_barrier();
      if (!role) {
        products(role, before, false, ka2, ka, vb);
        px_barrier();
        if (now) take();
      }
      products(role, now, false, ka1, ka, vb);
    } else {
      int slot = 0;
      for (int t = 0; t < steps; ++t) {
        __builtin_amdgcn_s_waitcnt(px_vm_wait(0));
        px_barrier();
        issue();
        const bool now = active_at(t);
        products(role, false, now, slot, slot, slot);
        if (now && !role) weights(t);
        px_barrier();
        if (now && role) slopes();
        px_barrier();
        if (now && !role) take();
        products(role, now, false, slot, slot, slot);
        slot = ring_next(slot, SA);
      }
    }
  };
  if (role)
    run(std::true_type{});
  else
    run(std::false_type{});

  unlift<T>(acc, lift);
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int q = q0 + 16 * n + r;
    back_store<T>(acc, n, q < nq, a.dq, a.part, (int64_t)a.Tq * a.Hq * D, part,
                  ((int64_t)(it.first + q) * a.Hq + head) * D + role * (D / 2), c, a.scale);
  }
}

// The parts of the split tiles added up, in their order: a workgroup has
// join_rows queries of a tile.
template <typename T, int D, int BQ>
__global__ __launch_bounds__(256) void k_attention_dq_join(AttnArgs a) {
  const AtPlace wg = at_place(a.Hq);
  const AtItem it = at_find(a.cu_q, a.B, a.Tq, BQ, wg.rank);
  if (it.seq < 0) return;
  int k_first, nk;
  at_rows(a.cu_k, a.B, a.Tk, it.seq, k_first, nk);
  const int wg0 = it.level * BQ;
  const int parts = at_parts(a, at_key_span(a, nk, nk - it.len, wg0, BQ, it.len, 32).steps);
  if (parts > 1)
    back_join<T, D>(a.part, (int64_t)a.Tq * a.Hq * D, parts, it.first, wg0 + join_rows(D) * (int)blockIdx.y, it.len,
                    a.Hq, wg.head, a.scale, a.dq);
}

// The queries that some key of a tile of `rows` from wg0 on sees, in steps of 32 of
// every head of the group.
__device__ __forceinline__ void query_range(const AttnArgs& a, int nq, int off, int first, int last, int& lo, int& hi) {
  lo = a.causal ? max(0, first - off) : 0;
  hi = a.window > 0 ? min(nq, last - off + a.window) : nq;
}
__device__ __forceinline__ AtSpan query_span(const AttnArgs& a, int nq, int nk, int wg0, int rows) {
  AtSpan s;
  query_range(a, nq, nk - nq, wg0, min(wg0 + rows, nk) - 1, s.lo, s.hi);
  s.lo &= ~31;
  s.steps = s.hi > s.lo ? (s.hi - s.lo + 31) / 32 : 0;
  return s;
}

// A workgroup has 16 NK keys of a key-value head per pair; A sums dv, B dk.
template <typename T, int D, int NK>
__global__ __launch_bounds__(kBackThreads, 2) void k_attention_dkv(AttnArgs a) {
  constexpr int SA = slots_a(D), SB = slots_b(D), S = SA + SB;
  constexpr int BK = 16 * NK * kPairs;
  constexpr int NI = D / 32, ND = D / 16;
  constexpr int kTile = at_tile_bytes<D>();
  constexpr int kAhead = 2;
  // steps that the loads are ahead, in the second phase
  constexpr int kAheadA = phases(D) ? SA - 2 : 1, kAheadB = SB - 1;
  using Feed = AtFeed<D, kPairs>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int role = wave / kPairs, place = wave % kPairs;

  const AtPlace wg = at_place(a.Hk);
  const int kvh = wg.head;
  const int index = __builtin_amdgcn_readfirstlane(wg.rank / a.tiles), tile = wg.rank - index * a.tiles;
  const AtItem it = at_find(a.cu_k, a.B, a.Tk, BK, tile);
  if (it.seq < 0) return;
  int q_first, nq;
  at_rows(a.cu_q, a.B, a.Tq, it.seq, q_first, nq);
  const int nk = it.len, off = nk - nq;
  const int wg0 = (it.tiles - 1 - it.level) * BK;  // the first keys are seen by the most queries
  const int k0 = wg0 + 16 * NK * place;
  int wlo, whi;
  query_range(a, nq, off, k0, min(k0 + 16 * NK, nk) - 1, wlo, whi);
  if (k0 >= nk) whi = 0;
  const AtSpan span = query_span(a, nq, nk, wg0, BK);
  const int per = max(span.steps, 1), lo = span.lo;  // steps of a head
  const AtPart part = at_part(a, span.steps * a.group, index);
  if (part.index >= part.of) return;
  const int steps = part.steps;
  const int top = lo + 32 * (per - 1);

  // A place in the steps: a head after the other, its queries from the last on.
  // (So all workgroups of a sequence that run together read the same tiles.)
  struct At {
    int head, q0;
  };
  auto onward = [&](At& x) {
    x.q0 -= 32;
    if (x.q0 < lo) {
      x.q0 = top;
      ++x.head;
    }
  };
  Feed feed;
  if (role)
    feed.init(static_cast<const unsigned char*>(a.dout) + (int64_t)q_first * a.Hq * D * 2, (int64_t)a.Hq * D * 2,
              place);
  else
    feed.init(static_cast<const unsigned char*>(a.q) + q_first * a.q_stride, a.q_stride, place);
  const int64_t head_bytes = role ? D * 2 : a.q_head;
  unsigned char* const ring = smem + (role ? SA * kTile : 0);
  const int heads = __builtin_amdgcn_readfirstlane(part.first / per);  // in front of the part
  const At begin{kvh * a.group + heads, top - 32 * (part.first - heads * per)};
  At next = begin;
  feed.seek(next.q0, nq, next.head * head_bytes);
  int load = 0, to = 0;
  auto issue = [&] {
    feed.issue(ring + to * kTile, load < steps);
    onward(next);
    if (next.q0 == top)
      feed.seek(top, nq, next.head * head_bytes);
    else
      feed.skip(-1);
    ++load;
    to = ring_next(to, role ? SB : SA);
  };
#pragma unroll
  for (int s = 0; s < (kAheadA > kAheadB ? kAheadA : kAheadB); ++s)
    if (s < (role ? kAheadB : kAheadA)) issue();

  u32x4_t rows[NK][NI];  // of k (A) or v
  f32x4_t acc[ND][NK];
  {
    const unsigned char* rp = role ? static_cast<const unsigned char*>(a.v) + kvh * a.v_head
                                   : static_cast<const unsigned char*>(a.k) + kvh * a.k_head;
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      at_load_row<NI>(rp, it.first + min(k0 + 16 * n + r, nk - 1), role ? a.v_stride : a.k_stride, rows[n]);
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
  }
  at_settle(rows);
  AtLane<D> ln;
  ln.init();
  // the exchange [place][lane]: p [tile][n], then (fp16) the powers of B's columns, for which
  // heads of 256 have no registers over the steps
  f32x4_t* const xp = reinterpret_cast<f32x4_t*>(smem + S * kTile) + place * 3 * NK * 64 + lane;
  float* const xl = reinterpret_cast<float*>(xp + 2 * NK * 64);
  constexpr bool kAway = kLift<T> && D == 256;
  static_assert(NK <= 4, "in a lane's 16 bytes");
  float lift[NK];
#pragma unroll
  for (int n = 0; n < NK; ++n) {
    lift[n] = kFirstLift;
    if (kAway && role) xl[n] = kFirstLift;
  }
  const uint32_t base = at_lds(smem);

  // lse or delta of a lane's eight queries; past the last query zeros
  struct Stats {
    u32x4_t v[2];
  };
  const float* sp = (role ? a.delta : a.lse) + q_first;
  auto fetch = [&](const At& x, bool any) {
    Stats st;
    const auto rsrc = make_rsrc(sp + (int64_t)x.head * a.Tq + x.q0, any ? (uint32_t)max(nq - x.q0, 0) * 4u : 0u);
#pragma unroll
    for (int u = 0; u < 2; ++u) st.v[u] = buf_ld16(rsrc, 32 * c, 16 * u);
    return st;
  };
  At at = begin;
  Stats st = fetch(at, steps > 0);
#pragma unroll
  for (int u = 0; u < 2; ++u) asm volatile("" : "+v"(st.v[u]));
  f32x4_t s[2][NK];
  u32x4_t p[NK];

  auto active_at = [&] { return at.q0 < whi && at.q0 + 32 > wlo; };
  // X: p times dout, or ds times the queries, of the step in qa1, gb1, and the
  // scores, or dout v^T, of that in qa, gb
  auto products = [&](auto role, bool sum, bool scores, int qa1, int gb1, int qa, int gb) {
    const uint32_t v = base + (role ? qa1 : SA + gb1) * kTile, w = base + (role ? SA + gb : qa) * kTile;
    u32x4_t next[kAhead];
    if (sum)
      at_accumulate<T, NI>(ln, v, p, acc, w, next);
    else
      at_scores_first<NI>(ln, w, next);
    if (scores) at_scores<T>(ln, w, rows, s, next);
  };
  auto pack = [&] {
#pragma unroll
    for (int n = 0; n < NK; ++n) p[n] = at_pack8<T>(s[0][n], s[1][n]);
  };
  auto weights = [&] {  // A
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // (one fma in place of the two has no register for its constants)
        const float lse2 = (__uint_as_float(st.v[u][i]) - kWeightLift<T> * kLn2) * kLog2e;
#pragma unroll
        for (int n = 0; n < NK; ++n)
          s[u][n][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][n][i], a.scale2, -lse2));
      }
    if (at.q0 + 32 > nq || k0 + 16 * NK > nk || (a.causal && k0 + 16 * NK - 1 > at.q0 + off) ||
        (a.window > 0 && k0 <= at.q0 + 31 + off - a.window)) {
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        // the queries low .. high of the step see the key
        const int key = k0 + 16 * n + r;
        const int low = a.causal ? key - off - at.q0 : 0;
        const int high = key >= nk ? -1 : (a.window > 0 ? min(nq, key - off + a.window) : nq) - 1 - at.q0;
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
    pack();
  };
  auto slope = [&](int n) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const f32x4_t w = xp[(u * NK + n) * 64];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[u][n][i] = w[i] * (s[u][n][i] - __uint_as_float(st.v[u][i]));
        if (kLift<T>) s[u][n][i] *= lift[n];
      }
    }
  };
  auto slopes = [&] {  // B
    if constexpr (kAway) {
      auto away = [&](auto N0) {
        constexpr int n = decltype(N0)::value;
        lift[n] = xl[n];
        slope(n);
        if (fit_slopes<n, n + 1>(s, acc, lift)) xl[n] = lift[n];
        p[n] = at_pack8<T>(s[0][n], s[1][n]);
      };
      away(std::integral_constant<int, 0>{});
      if constexpr (NK > 1) away(std::integral_constant<int, 1>{});
      static_assert(NK <= 2, "heads of 256");
    } else {
#pragma unroll
      for (int n = 0; n < NK; ++n) slope(n);
      if constexpr (kLift<T>) fit_slopes<0, NK>(s, acc, lift);
      pack();
    }
  };

  auto run = [&](auto role) {
    if constexpr (phases(D)) {
      int qa = 0, qa1 = SA - 1, gb = 0, gb1 = SB - 1;
      bool now = false;
      if (role) px_barrier();
      for (int t = 0; t < steps; ++t) {
        static_assert(kAheadA == kAheadB, "one wait for both");
        __builtin_amdgcn_s_waitcnt(px_vm_wait((kAheadA - 1) * Feed::kLoads));
        px_barrier();
        const bool before = now;
        now = active_at();
        __builtin_amdgcn_s_setprio(1);
        products(role, before, now, qa1, gb1, qa, gb);
        __builtin_amdgcn_s_setprio(0);
        px_barrier();
        if (now && !role) weights();
        if (now && role) slopes();
        onward(at);
        st = fetch(at, t + 1 < steps);  // in front of the loads, which then need not be waited for with it
        issue();
        qa1 = qa;
        gb1 = gb;
        qa = ring_next(qa, SA);
        gb = ring_next(gb, SB);
      }
      if (!role) px_barrier();
      products(role, now, false, qa1, gb1, qa, gb);
    } else {
      int slot = 0;
      for (int t = 0; t < steps; ++t) {
        __builtin_amdgcn_s_waitcnt(px_vm_wait(0));
        px_barrier();
        issue();
        const bool now = active_at();
        products(role, false, now, slot, slot, slot, slot);
        if (now && !role) weights();
        px_barrier();
        if (now && role) slopes();
        onward(at);
        st = fetch(at, t + 1 < steps);
        products(role, now, false, slot, slot, slot, slot);
        slot = ring_next(slot, SA);
      }
    }
  };
  if (role)
    run(std::true_type{});
  else
    run(std::false_type{});

#pragma unroll
  for (int n = 0; n < NK; ++n) lift[n] = !role ? 1.f : kAway ? xl[n] : lift[n];
  unlift<T>(acc, lift, 0x1p-12f);  // (kWeightLift)
  const int64_t plane = (int64_t)a.Tk * a.Hk * D;
  float* const parts = a.part + (role ? a.split * plane : 0);
#pragma unroll
  for (int n = 0; n < NK; ++n) {
    const int k = k0 + 16 * n + r;
    back_store<T>(acc, n, k < nk, role ? a.dk : a.dv, parts, plane, part, ((int64_t)(it.first + k) * a.Hk + kvh) * D, c,
                  role ? a.scale : 1.f);
  }
}

// As k_attention_dq_join: blockIdx.z 0 dv, 1 dk.
template <typename T, int D, int BK>
__global__ __launch_bounds__(256) void k_attention_dkv_join(AttnArgs a) {
  const AtPlace wg = at_place(a.Hk);
  const AtItem it = at_find(a.cu_k, a.B, a.Tk, BK, wg.rank);
  if (it.seq < 0) return;
  int q_first, nq;
  at_rows(a.cu_q, a.B, a.Tq, it.seq, q_first, nq);
  const int wg0 = (it.tiles - 1 - it.level) * BK;
  const int parts = at_parts(a, query_span(a, nq, it.len, wg0, BK).steps * a.group);
  const int64_t plane = (int64_t)a.Tk * a.Hk * D;
  const bool keys = blockIdx.z != 0;
  if (parts > 1)
    back_join<T, D>(a.part + (keys ? a.split * plane : 0), plane, parts, it.first,
                    wg0 + join_rows(D) * (int)blockIdx.y, it.len, a.Hk, wg.head, keys ? a.scale : 1.f,
                    keys ? a.dk : a.dv);
}

namespace {

template <typename T, int D, int N>
void launch_dq(const AttnArgs& a, hipStream_t s) {
  constexpr int BQ = 16 * N * kPairs;
  hipLaunchKernelGGL((k_attention_dq<T, D, N>), dim3((unsigned)(a.tiles * a.Hq * a.split)), dim3(kBackThreads),
                     back_lds(D, N), s, a);
  if (a.split > 1)
    hipLaunchKernelGGL((k_attention_dq_join<T, D, BQ>), dim3((unsigned)(a.tiles * a.Hq), BQ / join_rows(D)),
                       dim3(256), 0, s, a);
}
template <typename T, int D, int N>
void launch_dkv(const AttnArgs& a, hipStream_t s) {
  constexpr int BK = 16 * N * kPairs;
  hipLaunchKernelGGL((k_attention_dkv<T, D, N>), dim3((unsigned)(a.tiles * a.Hk * a.split)), dim3(kBackThreads),
                     back_lds(D, N), s, a);
  if (a.split > 1)
    hipLaunchKernelGGL((k_attention_dkv_join<T, D, BK>), dim3((unsigned)(a.tiles * a.Hk), BK / join_rows(D), 2),
                       dim3(256), 0, s, a);
}

template <typename T, int D>
hipError_t back(AttnArgs a, hipStream_t s) {
  constexpr int N = back_rows(D, false), L = back_rows(D, true);
  static_assert(back_lds(D, N) <= 160 * 1024 && attn_rows(kAttnDq, D) == attn_rows(kAttnDkv, D), "a CU's LDS");
  auto plan = [&](int kernel, int tokens) {
    const AttnSplit p = attn_split(kernel, a.B, a.Tq, a.Tk, a.Hq, a.Hk, a.D, a.window);
    a.split = p.split;
    a.chunk = p.chunk;
    a.low = p.low;
    a.tiles = tokens / attn_rows(kernel, D, p.low) + a.B + 1;
  };
  if (a.Tq > 0 && a.dq == nullptr)
    hipLaunchKernelGGL((k_attention_delta<T, D>), dim3((unsigned)(((int64_t)a.Tq * a.Hq + 63) / 64)), dim3(256), 0, s,
                       a);
  if (a.Tq > 0 && a.dq != nullptr) {
    plan(kAttnDq, a.Tq);
    a.low ? launch_dq<T, D, L>(a, s) : launch_dq<T, D, N>(a, s);
  }
  if (a.Tk > 0 && a.dk != nullptr) {
    plan(kAttnDkv, a.Tk);
    a.low ? launch_dkv<T, D, L>(a, s) : launch_dkv<T, D, N>(a, s);
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
