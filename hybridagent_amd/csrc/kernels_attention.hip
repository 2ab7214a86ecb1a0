// Attention over packed prompts: out = softmax(scale q k^T) v over the keys that
// a query sees, with grouped heads, sequences of any lengths packed one behind
// the other, causal masks and windows (include/w4a16moe.h, w4a16_attention).
#include <algorithm>
#include <climits>
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
// A loads the keys and B the values, each at the start of its Y, for S - 1 steps
// ahead: into the ring's slot that the step S before left.
constexpr int kGroup = 4, kWaves = 2 * kGroup;

// LDS slots of a ring, of steps of 32 KT keys
constexpr int fwd_slots(int D, int KT, int NQ) { return D == 256 || (D == 128 && NQ == 2) ? 3 : 2; }

}  // namespace

// Zero times a value that is not finite is not a number, so in a matrix product a key's value
// reaches the queries of its step that do not see it.  Only steps with hidden keys do that, so a
// column of a row can be wrong where one of the few hidden keys beside the row's own has such a
// value in it: these are looked for once per wavefront whose rows did not come out finite, and
// the columns summed again over the keys that the row sees.
template <typename T>
__device__ __forceinline__ bool not_finite(uint16_t x) {
  constexpr uint16_t kExponent = std::is_same_v<T, __bf16> ? 0x7F80 : 0x7C00;
  return (x & kExponent) == kExponent;
}
// a lane's E / 64 columns, side by side, of a row of values
template <int E>
struct LaneValues {
  static constexpr int kWords = E / 128 > 0 ? E / 128 : 1;
  typedef __attribute__((ext_vector_type(kWords))) uint32_t words_t;
  words_t w;
  __device__ __forceinline__ void load(const unsigned char* p) {
    if constexpr (E == 64)
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    else
      w = *reinterpret_cast<const words_t*>(p);
  }
  __device__ __forceinline__ uint16_t bits(int i) const { return (uint16_t)(w[i >> 1] >> (16 * (i & 1))); }
};
template <int E>
struct HiddenValues {
  int least[E / 64], most[E / 64];  // keys with such a value below the rows' keys, and above
};
// of the keys below .. below_end - 1 and above .. above_end - 1
template <typename T, int E>
__device__ __forceinline__ HiddenValues<E> hidden_values(const unsigned char* v, int64_t stride, int below,
                                                         int below_end, int above, int above_end, int at) {
  constexpr int VE = E / 64;
  const unsigned char* const p = v + 2 * (at + VE * (int)opaque(threadIdx.x & 63));
  HiddenValues<E> h;
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    h.least[i] = INT_MAX;
    h.most[i] = -1;
  }
  LaneValues<E> x;
#pragma unroll 4
  for (int key = below; key < below_end; ++key) {
    x.load(p + key * stride);
#pragma unroll
    for (int i = 0; i < VE; ++i) h.least[i] = not_finite<T>(x.bits(i)) ? min(h.least[i], key) : h.least[i];
  }
#pragma unroll 4
  for (int key = above; key < above_end; ++key) {
    x.load(p + key * stride);
#pragma unroll
    for (int i = 0; i < VE; ++i) h.most[i] = not_finite<T>(x.bits(i)) ? max(h.most[i], key) : h.most[i];
  }
  return h;
}
// A row to sum again: the keys from .. to that it sees, its maximum.
struct AgainRow {
  const unsigned char* q;
  int from, to;
  float m;
};
template <int E>
__device__ __forceinline__ bool hidden_hits(const HiddenValues<E>& h, const AgainRow& r, int i) {
  return h.least[i] < r.from || h.most[i] > r.to;
}
constexpr int kAgainRows = 4;
// The columns of kAgainRows rows with a hidden value, over the keys that each sees, from the last
// on in blocks of 64.  Ends where all of them are not finite by keys that their rows see, so
// that values that are not finite throughout cost a block.  Rows go together for the loads'
// sake (8192 keys of heads of 512, a block: one row 8.4 us, four 23).  store(row, column, sum).
template <typename T, int D, int E, typename Store>
__device__ __forceinline__ void attention_again(const AttnArgs& a, const HiddenValues<E>& hidden,
                                                const AgainRow (&rows)[kAgainRows], const unsigned char* k,
                                                const unsigned char* v, int at, const Store& store) {
  const int lane = (int)opaque(threadIdx.x & 63);  // (no register is kept for what comes of it over the steps)
  // L lanes have a key's row in turn, and lane i + L j of a block the key 64 / L i + j in the end;
  // C, U: loads of keys, of values together
  constexpr int VE = E / 64, L = D / 8, C = 8, U = 16, R = kAgainRows;
  float acc[R][VE];
  u32x4_t x[R];
  int from = INT_MAX, to = -1;
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int i = 0; i < VE; ++i) acc[r][i] = 0.f;
    x[r] = ld16(rows[r].q + 16 * (lane % L));
    if (rows[r].from <= rows[r].to) {
      from = min(from, rows[r].from);
      to = max(to, rows[r].to);
    }
  }
  const unsigned char* const lowest = k + (to < 0 ? 0 : from) * a.k_stride + 16 * (lane % L);
  const int64_t step = 64 / L * a.k_stride;
  for (int last = to; last >= from; last -= 64) {
    const int n = min(last - from + 1, 64);
    float p[R];
#pragma unroll
    for (int r = 0; r < R; ++r) p[r] = 0.f;
    const unsigned char* const first = lowest + (last - from - lane / L) * a.k_stride;
    for (int i0 = 0; i0 < L; i0 += C) {
      u32x4_t y[C];
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const unsigned char* const key = first - (i0 + i) * step;
        y[i] = ld16(key < lowest ? lowest : key);
      }
#pragma unroll
      for (int i = 0; i < C; ++i)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float s = 0.f;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            s = __builtin_fmaf(at_lo<T>(x[r][w]), at_lo<T>(y[i][w]), s);
            s = __builtin_fmaf(at_hi<T>(x[r][w]), at_hi<T>(y[i][w]), s);
          }
          s = at_sum_over<L>(s);
          p[r] = lane % L == i0 + i ? s : p[r];
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[r], a.scale2, -rows[r].m));
    const unsigned char* const columns = v + 2 * (at + VE * lane);
    for (int j0 = 0; j0 < n; j0 += U) {
      LaneValues<E> y[U];
#pragma unroll
      for (int j = 0; j < U; ++j) y[j].load(columns + max(last - j0 - j, from) * a.v_stride);
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int of = j0 + j, key = last - of, owner = of % (64 / L) * L + of / (64 / L);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p[r]), owner));
          const bool seen = key >= rows[r].from && key <= rows[r].to;
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            const float sum = __builtin_fmaf(w, at_lo<T>(y[j].bits(i)), acc[r][i]);
            acc[r][i] = seen ? sum : acc[r][i];
          }
        }
      }
    }
    bool more = false;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < VE; ++i) more |= hidden_hits(hidden, rows[r], i) && __builtin_fabsf(acc[r][i]) < INFINITY;
    if (__ballot(more) == 0) break;
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (hidden_hits(hidden, rows[r], i)) store(r, at + VE * lane + i, acc[r][i]);
}

// Where a part of a split tile leaves a query's sums and (m, l), and the query's
// place in out and lse: [split][Tq][Hq][D], then [split][Hq][Tq].
__device__ __forceinline__ float* fwd_part(const AttnArgs& a, int part, int64_t token, int head) {
  return a.part + (((int64_t)part * a.Tq + token) * a.Hq + head) * a.D;
}
__device__ __forceinline__ float2* fwd_stats(const AttnArgs& a, int part, int64_t token, int head) {
  return reinterpret_cast<float2*>(a.part + (int64_t)a.split * a.Tq * a.Hq * a.D) +
         ((int64_t)part * a.Hq + head) * a.Tq + token;
}

// Bound, heads of 256 and 512: the matrix units between the barriers.  A phase X of heads of 256 takes
// 1450 cycles, of which 1024 are its 64 matrix instructions (its LDS reads as many,
// free of bank conflicts; wider than two tiles of queries a wavefront there are no
// registers); Y hides behind the other group's X.  Of 64 and 128 Y is the longer: a score
// costs an fma, a maximum, an exponential, a sum and half a packing there, whatever D is,
// and the matrix units are busy 0.30 and 0.45 of the CUs' cycles (256: 0.52).
// 2 x 4096 tokens, 16 heads, 8 key-value heads: heads of 64 97-102 us (680 TFLOP/s of the
// pairs seen), 128 132-138 (1030), 256 225-235 (1190), 512 502-524 (1070); a product of
// 8192^3 reaches 1373.  A window of 1024 keys: 67, 88, 148, 288 us; all keys seen: 168,
// 242, 412, 940.  fp16: 110, 145, 248, 530.
//
// A workgroup has 16 NQ queries of a head per wavefront; PAIR: per pair of
// wavefronts of a group, each with half of D: of the scores' sum, whose halves
// they exchange through LDS between the phases, and of the output's columns.
// (Heads of 512: a wavefront's registers hold 16 queries' output and the queries,
// and every operand read from LDS would feed one matrix instruction.)
// SPLIT: a tile's steps may have several parts.
template <typename T, int D, int NQ, int KT, bool PAIR, bool SPLIT>
__global__ __launch_bounds__(64 * kWaves, NQ == 1 && D <= 128 ? 4 : 2) void k_attention(AttnArgs a) {
  constexpr int S = fwd_slots(D, KT, NQ);
  constexpr int kHalves = PAIR ? 2 : 1;
  constexpr int BQ = 16 * NQ * kWaves / kHalves;
  constexpr int NI = D / 32 / kHalves, ND = D / 16 / kHalves;
  constexpr int kTile = at_tile_bytes<D>(), kStepBytes = KT * kTile, kKeys = 32 * KT;
  constexpr int kAhead = 2;
  using Feed = AtFeed<D, kGroup>;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool second = wave >= kGroup;  // group B
  const int half = PAIR ? wave & 1 : 0;

  const AtPlace at = at_place(a.Hq);
  const int index = SPLIT ? __builtin_amdgcn_readfirstlane(at.rank / a.tiles) : 0, tile = at.rank - index * a.tiles;
  const AtItem it = at_find(a.cu_q, a.B, a.Tq, BQ, tile);
  if (it.seq < 0) return;
  int k_first, nk;
  at_rows(a.cu_k, a.B, a.Tk, it.seq, k_first, nk);
  const int nq = it.len, off = nk - nq;
  const int wg0 = it.level * BQ;
  const int q0 = wg0 + 16 * NQ * (wave / kHalves);

  int wlo, whi;
  at_seen_keys(a, nk, off, q0, min(q0 + 16 * NQ, nq) - 1, wlo, whi);
  if (q0 >= nq) whi = 0;
  const AtSpan span = at_key_span(a, nk, off, wg0, BQ, nq, kKeys);
  const AtPart part = SPLIT ? at_part(a, span.steps, index) : AtPart{0, 1, 0, span.steps};
  if (part.index >= part.of) return;
  const int lo = span.lo + kKeys * part.first, hi = span.hi, steps = part.steps;

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
  feed.seek(lo, hi);
  unsigned char* const ring = smem + (second ? S * kStepBytes : 0);
  auto issue = [&](int slot, int t) {
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      feed.issue(ring + slot * kStepBytes + k * kTile, t < steps);
      feed.skip(1);
    }
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) issue(s, s);

  u32x4_t qf[NQ][NI];
  float m[NQ], l[NQ];
  f32x4_t acc[ND][NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    at_load_row<NI>(static_cast<const unsigned char*>(a.q) + at.head * a.q_head + half * D,
                    it.first + min(q0 + 16 * n + r, nq - 1), a.q_stride, qf[n]);
    m[n] = 0.f;
    l[n] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  at_settle(qf);
  AtLane<D> ln;
  ln.init();
  if constexpr (PAIR) {
    ln.half_rows(half);
    ln.half_cols(half);
  }
  // the pairs' exchange: [wave][tile][n][lane]
  f32x4_t* const mine = reinterpret_cast<f32x4_t*>(smem + 2 * S * kStepBytes) + wave * 2 * KT * NQ * 64 + lane;
  const f32x4_t* const other = mine + (half ? -1 : 1) * 2 * KT * NQ * 64;
  const uint32_t base = at_lds(smem);

  f32x4_t s[KT][2][NQ];
  u32x4_t p[KT][NQ];
  // X: the weights of a step times its values, in slot `from`, and the scores of one
  // whose keys are in slot `of`
  auto products = [&](bool sum, bool scores, int from, int of) {
    u32x4_t next[kAhead];
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      const uint32_t v = base + (S + from) * kStepBytes + k * kTile, w = base + of * kStepBytes + k * kTile;
      if (sum)
        at_accumulate<T, NI>(ln, v, p[k], acc, w, next);
      else
        at_scores_first<NI>(ln, w, next);
      if (scores) at_scores<T>(ln, w, qf, s[k], next);
    }
  };
  bool active = false;  // the last step had keys that the wavefront's queries see
  if (second) px_barrier();
  int slot = 0, last = S - 1;  // of step t, of the step before (and of the next to load)
  for (int t = 0; t < steps; ++t) {
    if (!second) __builtin_amdgcn_s_waitcnt(px_vm_wait((S - 2) * KT * Feed::kLoads));
    px_barrier();
    const int key0 = lo + kKeys * t;
    const bool before = active;
    active = key0 < whi && key0 + kKeys > wlo;
    __builtin_amdgcn_s_setprio(1);
    products(before, active, last, slot);
    __builtin_amdgcn_s_setprio(0);
    if (active) {
      if constexpr (PAIR) {
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int n = 0; n < NQ; ++n) mine[((k * 2 + u) * NQ + n) * 64] = s[k][u][n];
      }
    }
    if (second) __builtin_amdgcn_s_waitcnt(px_vm_wait((S - 2) * KT * Feed::kLoads));
    px_barrier();
    issue(last, t + S - 1);
    last = slot;
    slot = slot == S - 1 ? 0 : slot + 1;
    if (!active) continue;
    if constexpr (PAIR) {
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[k][u][n] += other[((k * 2 + u) * NQ + n) * 64];
    }
    // some query does not see some key
    if (key0 + kKeys > nk || (a.causal && key0 + kKeys - 1 > q0 + off) ||
        (a.window > 0 && key0 <= min(q0 + 16 * NQ, nq) - 1 + off - a.window)) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int q = q0 + 16 * n + r + off;
        const int to = a.causal ? min(nk - 1, q) : nk - 1;
        const int from = a.window > 0 ? q - a.window + 1 : 0;
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = key0 + 32 * k + 8 * c + 4 * u + i;
              s[k][u][n][i] = key <= to && key >= from ? s[k][u][n][i] : -INFINITY;
            }
      }
    }
    // The exponents, from the running maximum as it is.  It moves where one is
    // above kOver, so that the weights stay below 2^kOver; and to the first
    // that a query sees (a lane without a weight so far asks).
    float top[NQ];
    bool over = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      top[n] = -INFINITY;
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[k][u][n][i] = __builtin_fmaf(s[k][u][n][i], a.scale2, -m[n]);
            top[n] = fmaxf(top[n], s[k][u][n][i]);
          }
      over |= top[n] > (l[n] == 0.f ? -INFINITY : AtWeight<T>::kOver);
    }
    if (__any(over)) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const float t = at_max_over_c(top[n]) - AtWeight<T>::kTop;
        const bool first = at_sum_over_c(l[n]) == 0.f;
        const float up = t > (first ? -INFINITY : 0.f) ? t : 0.f;
        // the first seen may lie far below zero: nothing is summed yet, and 0 x 2^-up would not be a number
        const float f = first ? 1.f : __builtin_amdgcn_exp2f(-up);
        m[n] += up;
        l[n] *= f;
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
          for (int u = 0; u < 2; ++u) s[k][u][n] -= up;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d][n] *= f;
      }
    }
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[k][u][n][i] = __builtin_amdgcn_exp2f(s[k][u][n][i]);
            l[n] += s[k][u][n][i];
          }
        p[k][n] = at_pack8<T>(s[k][0][n], s[k][1][n]);
      }
  }
  if (!second) px_barrier();
  products(active, false, last, slot);

  unsigned char* const out = static_cast<unsigned char*>(a.out) + ((int64_t)it.first * a.Hq + at.head) * (D * 2);
  const int64_t out_row = (int64_t)a.Hq * D * 2;
  const bool whole = !SPLIT || part.of == 1;
  unsigned long long odd[NQ];  // lanes with a result that is not finite
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int q = q0 + 16 * n + r;
    l[n] = at_sum_over_c(l[n]);
    const float f = !whole ? 1.f : l[n] != 0.f ? 1.0f / l[n] : at_sees(a, nk, off, q) ? NAN : 0.f;
    if (c == 0 && half == 0 && q < nq) {
      if (!whole)
        *fwd_stats(a, part.index, it.first + q, at.head) = float2{l[n] == 0.f ? -INFINITY : m[n], l[n]};
      else if (a.lse != nullptr)
        a.lse[(int64_t)at.head * a.Tq + it.first + q] = (m[n] + __builtin_amdgcn_logf(l[n])) * kLn2;
    }
    float zero = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      acc[d][n] *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i) zero = __builtin_fmaf(acc[d][n][i], 0.f, zero);
    }
    if (whole) {
      unsigned char* o = out + q * out_row + half * D + 2 * at_pair_column(c);
#pragma unroll
      for (int d = 0; d < ND; d += 2) {
        const u32x4_t v = at_pair<T>(acc[d][n], acc[d + 1][n]);
        if (q < nq) *reinterpret_cast<u32x4_t*>(o + 32 * d) = v;
      }
    } else if (q < nq) {
      float* o = fwd_part(a, part.index, it.first + q, at.head) + half * (D / 2) + 4 * c;
#pragma unroll
      for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4_t*>(o + 16 * d) = acc[d][n];
    }
    odd[n] = __ballot(q < nq && zero != 0.f && l[n] == l[n]);  // a sum that is not: a seen key's score
  }
  if (!a.causal) return;
  bool again = false;
#pragma unroll
  for (int n = 0; n < NQ; ++n) again |= odd[n] != 0;
  if (!again) return;
  __builtin_amdgcn_s_waitcnt(px_vm_wait(0));  // the rows' first stores are done
  const int kvh = at.head / a.group;
  const unsigned char* const qp = static_cast<const unsigned char*>(a.q) + at.head * a.q_head;
  const unsigned char* const kp = static_cast<const unsigned char*>(a.k) + k_first * a.k_stride + kvh * a.k_head;
  const unsigned char* const vp = static_cast<const unsigned char*>(a.v) + k_first * a.v_stride + kvh * a.v_head;
  // the keys that the rows' last and first see, and of the steps that the wavefront took
  const int begin = max(lo, wlo - kKeys + 1), end = min(min(lo + kKeys * steps, hi), whi + kKeys - 1);
  const int q_last = min(q0 + 16 * NQ, nq) - 1;
  const int below = a.window > 0 ? min(end, q_last + off - a.window + 1) : begin, above = max(begin, q0 + off + 1);
  const HiddenValues<D / kHalves> hidden =
      hidden_values<T, D / kHalves>(vp, a.v_stride, begin, below, above, end, half * (D / 2));
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    unsigned long long left = (odd[n] | odd[n] >> 16 | odd[n] >> 32 | odd[n] >> 48) & 0xFFFFull;
    while (left != 0) {
      AgainRow rows[kAgainRows];
      int q[kAgainRows], r = 0;
      float sum[kAgainRows];
      while (left != 0 && r < kAgainRows) {
        const int i = __ffsll(left) - 1;
        left &= left - 1;
        const int query = q0 + 16 * n + i;
        const AgainRow row{qp + (it.first + query) * a.q_stride, max(lo, a.window > 0 ? query + off - a.window + 1 : 0),
                           min(lo + kKeys * steps, min(nk, query + off + 1)) - 1,
                           __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(m[n]), i))};
        bool hit = false;
#pragma unroll
        for (int j = 0; j < D / kHalves / 64; ++j) hit |= hidden_hits(hidden, row, j);
        if (__ballot(hit) == 0) continue;
        // (the rest of the places: this one once more)
        const float l1 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(l[n]), i));
#pragma unroll
        for (int j = 0; j < kAgainRows; ++j)
          if (j >= r) {
            rows[j] = row;
            q[j] = query;
            sum[j] = l1;
          }
        ++r;
      }
      if (r == 0) break;
      attention_again<T, D, D / kHalves>(a, hidden, rows, kp, vp, half * (D / 2), [&](int j, int d, float v) {
        if (whole)
          *reinterpret_cast<uint16_t*>(out + q[j] * out_row + 2 * d) =
              (uint16_t)at_pack2<T>(sum[j] == 0.f && !at_sees(a, nk, off, q[j]) ? 0.f : v / sum[j], 0.f);
        else
          fwd_part(a, part.index, it.first + q[j], at.head)[d] = v;
      });
    }
  }
}

constexpr int kAttnJoin = 4;

// The parts of the split tiles put together: a workgroup has kAttnJoin 1024 / D
// queries of a tile, whose loads are under way together.
template <typename T, int D, int BQ, int kKeys>
__global__ __launch_bounds__(256) void k_attention_join(AttnArgs a) {
  constexpr int L = D / 4;
  const AtPlace at = at_place(a.Hq);
  const AtItem it = at_find(a.cu_q, a.B, a.Tq, BQ, at.rank);
  if (it.seq < 0) return;
  int k_first, nk;
  at_rows(a.cu_k, a.B, a.Tk, it.seq, k_first, nk);
  const int nq = it.len, wg0 = it.level * BQ;
  const int parts = at_parts(a, at_key_span(a, nk, nk - nq, wg0, BQ, nq, kKeys).steps);
  if (parts == 1) return;
  constexpr int R = kAttnJoin;
  const int d = 4 * (threadIdx.x % L), q0 = wg0 + R * (256 / L) * blockIdx.y + threadIdx.x / L;
  if (q0 >= nq) return;
  int64_t token[R];
  float top[R], l[R];
  f32x4_t v[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    token[i] = it.first + min(q0 + 256 / L * i, nq - 1);
    top[i] = -INFINITY;
    l[i] = 0.f;
    v[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll 4
  for (int p = 0; p < parts; ++p)
#pragma unroll
    for (int i = 0; i < R; ++i) top[i] = fmaxf(top[i], fwd_stats(a, p, token[i], at.head)->x);
#pragma unroll 2
  for (int p = 0; p < parts; ++p)
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float2 s = *fwd_stats(a, p, token[i], at.head);
      const float f = __builtin_amdgcn_exp2f(s.x - (top[i] == -INFINITY ? 0.f : top[i]));
      l[i] += s.y * f;
      v[i] += *reinterpret_cast<const f32x4_t*>(fwd_part(a, p, token[i], at.head) + d) * f;
    }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (q0 + 256 / L * i >= nq) break;
    const float f = l[i] != 0.f ? 1.0f / l[i] : at_sees(a, nk, nk - nq, q0 + 256 / L * i) ? NAN : 0.f;
    *reinterpret_cast<u32x2_t*>(static_cast<unsigned char*>(a.out) + ((token[i] * a.Hq + at.head) * D + d) * 2) =
        u32x2_t{at_pack2<T>(v[i][0] * f, v[i][1] * f), at_pack2<T>(v[i][2] * f, v[i][3] * f)};
    // (no key at all: log2 0 is the least)
    if (a.lse != nullptr && d == 0)
      a.lse[(int64_t)at.head * a.Tq + token[i]] =
          ((top[i] == -INFINITY ? 0.f : top[i]) + __builtin_amdgcn_logf(l[i])) * kLn2;
  }
}

namespace {

template <typename T, int D, int NQ, int KT, bool PAIR>
hipError_t fwd(AttnArgs a, hipStream_t s) {
  a.tiles = a.Tq / (16 * NQ * kWaves / (PAIR ? 2 : 1)) + a.B + 1;
  constexpr int lds = 2 * fwd_slots(D, KT, NQ) * KT * at_tile_bytes<D>() + (PAIR ? kWaves * 2 * KT * NQ * 64 * 16 : 0);
  static_assert(lds <= 160 * 1024, "a CU's LDS");
  constexpr int BQ = 16 * NQ * kWaves / (PAIR ? 2 : 1);
  static_assert(BQ == attn_rows(kAttnForward, D, NQ == 1), "attn_split's tiles");
  static_assert(32 * KT == attn_keys(kAttnForward, D), "attn_split's steps");
  const dim3 grid((unsigned)(a.tiles * a.Hq * a.split));
  if (a.split == 1) {
    hipLaunchKernelGGL((k_attention<T, D, NQ, KT, PAIR, false>), grid, dim3(64 * kWaves), lds, s, a);
  } else if constexpr (!PAIR || NQ == 1) {
    hipLaunchKernelGGL((k_attention<T, D, NQ, KT, PAIR, true>), grid, dim3(64 * kWaves), lds, s, a);
    hipLaunchKernelGGL((k_attention_join<T, D, BQ, 32 * KT>),
                       dim3((unsigned)(a.tiles * a.Hq), BQ * D / 1024 / kAttnJoin), dim3(256), 0, s, a);
  } else {
    return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

template <typename T>
hipError_t fwd_type(const AttnArgs& a, bool low, hipStream_t s) {
  switch (a.D) {
    case 64: return low ? fwd<T, 64, 1, 2, false>(a, s) : fwd<T, 64, 2, 2, false>(a, s);
    case 128: return low ? fwd<T, 128, 1, 2, false>(a, s) : fwd<T, 128, 2, 2, false>(a, s);
    case 256: return low ? fwd<T, 256, 1, 1, false>(a, s) : fwd<T, 256, 2, 1, false>(a, s);
    case 512: return low ? fwd<T, 512, 1, 1, true>(a, s) : fwd<T, 512, 2, 1, true>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

// Tiles with few heads or tokens leave most CUs idle, and a tile's steps follow one
// another: they are cut so that there are about two workgroups per CU, of kAttnChunk
// steps at least (a part costs some 10 us of its own: its start, its sums to memory and
// back).  4096 tokens, 8 heads and one key-value head of 128: dk and dv 1600 -> 217 us,
// dq 182 -> 130, forward 116 -> 82; 2000 tokens, 4 heads of 256, a training step 581 ->
// 131 us, with 8 steps at least 172, with 16 138.  The host knows the sequences' number and
// sum, not their lengths: tiles and chunks go by the mean, and a long sequence among short
// ones has theirs.  Above 64 sequences, where at_find goes round the offsets, none are cut:
// that was not tried.
AttnSplit attn_split(int kernel, int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D, int64_t window) {
  AttnSplit r{false, 1, 1, 0};
  const bool dkv = kernel == kAttnDkv;
  const int64_t heads = dkv ? Hk : Hq, each = dkv ? Hq / Hk : 1;
  const int64_t T = dkv ? Tk : Tq, other = dkv ? Tq : Tk;
  // Smaller tiles where the others leave CUs idle (forward: 180 tokens of 16 heads of
  // 256 19 -> 14 us).  Backward, by the sequences' length: of 128, in 64 rows two
  // workgroups share a CU, which up to 2048 tokens outweighs the operands they read
  // twice (8 x 1024 tokens, 8 heads, dq 90 -> 56 us, dk and dv 112 -> 72; 4096 tokens
  // 108 -> 121 and 143 -> 142); of 256 they do not fit, and a step's latency alone
  // speaks for it (8 x 256 tokens 31 -> 27 and 44 -> 37; 2 x 1024 44 -> 54 and 59 -> 64).
  const int64_t even = other / std::max<int64_t>(B, 1), length = window > 0 ? std::min(even, window) : even;
  r.low = kernel == kAttnForward ? (T / attn_rows(kernel, (int)D) + B + 1) * heads <= attn_low(D)
                                 : length <= (D == 128 ? 2048 : D == 256 ? 256 : 0);
  const int64_t rows = attn_rows(kernel, (int)D, r.low), keys = attn_keys(kernel, (int)D);
  if (B <= 0 || B > 64 || T <= 0 || other <= 0) return r;
  const int64_t tiles = T / rows + B + 1;
  // sequences of one length: their tiles, and a tile's steps
  const int64_t like = ((T / B + rows - 1) / rows) * B;
  auto steps = [&](int64_t n) {
    const int64_t seen = window > 0 && window < n ? std::min(n, window + rows) : n;
    return ((seen + keys - 1) / keys + 1) * each;
  };
  const int64_t work = like * heads * steps(other / B);
  const int64_t chunk = std::max<int64_t>(kAttnChunk, work / kAttnParts);
  const int64_t split =
      std::min<int64_t>({kAttnMostParts, steps(other) / chunk, 2 * kAttnParts / (tiles * heads)});
  if (split < 2) return r;
  r.split = (int)split;
  r.chunk = (int)chunk;
  r.floats = dkv ? (size_t)(2 * split * Tk * Hk * D)
                 : (size_t)(split * Tq * Hq * (D + (kernel == kAttnForward ? 2 : 0)));
  return r;
}

hipError_t launch_attention(int dtype, const AttnArgs& a, hipStream_t s) {
  return dtype == 0 ? fwd_type<__bf16>(a, a.low, s) : fwd_type<_Float16>(a, a.low, s);
}

}  // namespace w4a16
