// Attention of one new token per sequence over the paged key-value cache
// (include/w4a16moe.h, w4a16_decode_attention): the cache read once, at the
// memory's rate.
//
// The keys of a sequence that the token sees are cut into steps of 128.  Where there
// are few by the table's width, a workgroup has all of a (sequence, head).  Else the
// steps of all sequences and key-value heads (16 queries of a group at most)
// are one row, dealt out evenly to the workgroups, whatever the lengths.  A
// workgroup's part of a (sequence, head)'s steps is a piece: if it is all of them
// its result is the output, else it goes to the workspace, two pieces a
// workgroup at most, and k_decode_join adds them up in their order.  The cut
// depends on the lengths alone.
//
// A wavefront takes 32 keys of a step by itself, straight from memory into the
// operands of the matrix instructions, with no LDS between: a key's row is the
// first operand of the scores as it lies (64 bytes of 16 rows a load), and of the
// values a lane loads the 8 x 8 block of its eight keys and eight columns, 256
// bytes of a row per load, which 32 byte permutations turn around in its
// registers.
//
// Bound: the cache's bytes.  64 sequences of 4000 keys, 8 key-value heads of 128: 183
// us, 5.7 TB/s; of 2000 keys of 256 180 us, 5.8 (reads alone; a copy reaches 4.95); of
// 64 x 4000 keys of 64 98 us, 5.4.  A few sequences: the first loads, one after the
// other (length, page, keys), 5 us, and the join's launch.
#include <algorithm>
#include <type_traits>

#include "attention.hpp"

namespace w4a16 {

namespace {

constexpr int kDaWaves = 4;
constexpr int kDaStep = 32 * kDaWaves;  // keys

// the keys first .. len - 1 that a sequence's token sees, in steps from base on
struct DaSeq {
  int len, first, base, steps;
  bool over;  // longer than its row of the table
};
__device__ __forceinline__ DaSeq da_seq(const DecodeAttnArgs& a, int b) {
  DaSeq s;
  const int n = a.lengths[b], cap = a.width << a.page_log2;
  s.over = n > cap;
  s.len = max(min(n, cap), 0);
  s.first = a.window > 0 ? max(s.len - a.window, 0) : 0;
  s.base = s.first & ~31;
  s.steps = max((s.len - s.base + kDaStep - 1) / kDaStep, 1);  // one without keys: it writes the zeros
  return s;
}

// steps in front of sequence b (all of them: b = B), of one head
__device__ __forceinline__ int da_before(const DecodeAttnArgs& a, int b) {
  int sum = 0;
  for (int i = threadIdx.x & 63; i < b; i += 64) sum += da_seq(a, i).steps;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
  return sum;
}

// the first step of workgroup g's of `total`
__device__ __forceinline__ int da_start(int g, int groups, int total) {
  return (int)((int64_t)total * g / groups);
}

}  // namespace

template <typename T, int D>
__global__ __launch_bounds__(64 * kDaWaves, D == 512 ? 1 : 2) void k_decode_attention(DecodeAttnArgs a) {
  constexpr int VW = D >= 128 ? 8 : 4;    // columns of a lane's block of values
  constexpr int NB = D / (16 * VW);       // blocks
  constexpr int VD = VW / 2;              // dwords of a block's row
  constexpr bool kEarly = D < 256;
  __shared__ float sm[kDaWaves][16], sl[kDaWaves][16];
  extern __shared__ __align__(16) float so[];  // [kDaWaves][D * 16]
  const int lane = threadIdx.x & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int gt = (a.group + 15) / 16;  // tiles of a group's queries
  const int units = a.Hk * gt;

  // the workgroup's steps pos .. end - 1, the sequence of the first, and the steps
  // `at` in front of that
  int pos, end, b = 0, at = 0;
  auto deal = [&](int total) {
    const int groups = min(a.groups, total);  // each has a step at least
    if ((int)blockIdx.x >= groups) return false;
    pos = da_start(blockIdx.x, groups, total);
    end = da_start(blockIdx.x + 1, groups, total);
    return true;
  };
  if (a.whole) {
    b = (int)blockIdx.x / units;
    const int steps = da_seq(a, b).steps;
    pos = ((int)blockIdx.x - b * units) * steps;
    end = pos + steps;
  } else if (a.B > 64 && !deal(da_before(a, a.B) * units)) {
    return;
  }
  for (int base = 0; !a.whole && base < a.B; base += 64) {
    const int n = base + lane < a.B ? da_seq(a, base + lane).steps * units : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o);
      if (lane >= o) sum += v;
    }
    const int all = __builtin_amdgcn_readlane(sum, 63);
    if (a.B <= 64 && !deal(all)) return;
    if (pos < at + all) {
      const int i = __ffsll((unsigned long long)__ballot(at + sum > pos)) - 1;
      b = base + i;
      at += __builtin_amdgcn_readlane(sum - n, i);
      break;
    }
    at += all;
  }
  const int begin = pos;

  while (pos < end) {
    const DaSeq seq = da_seq(a, b);
    const int unit = (pos - at) / seq.steps;
    const int s0 = pos - at - unit * seq.steps, s1 = min(seq.steps, s0 + end - pos);
    const int hk = unit / gt, q_first = (unit - hk * gt) * 16, q_n = min(a.group - q_first, 16);
    const int head0 = hk * a.group + q_first;

    const int64_t in_page = (int64_t)hk * (D * 2) << a.page_log2;
    const unsigned char* kp = static_cast<const unsigned char*>(a.kc) + in_page;
    const unsigned char* vp = static_cast<const unsigned char*>(a.vc) + in_page;
    const int32_t* row = a.table + (int64_t)b * a.width;
    const int mask = (1 << a.page_log2) - 1;
    // A lane's keys are held to the ones that are seen (those beside them may lie
    // in pages that are another's by now, and hold anything): a group of eight
    // keys, all of one page, has its page or, with none seen, the nearest's.
    auto hold = [&](int key) { return min(max(key, seq.first), seq.len - 1); };
    // the pages of a lane's eight keys as rows of the scores (k) and of the values (v)
    struct Pages {
      int k, v;
    };
    auto pages = [&](int key0) {
      return Pages{row[hold(key0 + 8 * (r >> 2)) >> a.page_log2], row[hold(key0 + 8 * c) >> a.page_log2]};
    };
    u32x4_t kf[2][D / 32];
    auto keys = [&](int key0, int page) {
      const unsigned char* p = kp + (page < 0 || page >= a.pages ? 0 : page) * a.k_page;
#pragma unroll
      for (int t = 0; t < 2; ++t)
        at_load_row<D / 32>(p, hold(key0 + 8 * (r >> 2) + 4 * t + (r & 3)) & mask, D * 2, kf[t]);
    };

    // The wavefront's keys of a step are key0 ..; the next ones' pages are read a step
    // ahead.  kEarly: their rows too, once the scores are done with these (heads of
    // 256: two wavefronts of a SIMD cover for each other instead, without the room).
    int key0 = seq.base + s0 * kDaStep + 32 * wave;
    const int stop = min(seq.len, seq.base + s1 * kDaStep);
    Pages now{0, 0}, next{0, 0};
    if (key0 < stop) {
      now = pages(key0);
      if (key0 + kDaStep < stop) next = pages(key0 + kDaStep);
      if (kEarly) keys(key0, now.k);
    }
    u32x4_t qf[D / 32];
    at_load_row<D / 32>(static_cast<const unsigned char*>(a.q) + (int64_t)(head0 + min(r, q_n - 1)) * a.q_head, b,
                        a.q_stride, qf);

    float m = 0.f, l = 0.f;
    f32x4_t acc[NB][VW];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int e = 0; e < VW; ++e) acc[j][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    for (; key0 < stop; key0 += kDaStep) {
      if (!kEarly) keys(key0, now.k);
      const bool bad = seq.over || now.v < 0 || now.v >= a.pages;
      uint32_t vf[NB][8][VD];
      {
        const unsigned char* q = vp + (bad ? 0 : now.v) * a.v_page + r * (2 * VW);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const unsigned char* p = q + (int64_t)(hold(key0 + 8 * c + i) & mask) * (D * 2);
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            if constexpr (VW == 8) {
              const u32x4_t v = ld16(p + 256 * j);
#pragma unroll
              for (int w = 0; w < 4; ++w) vf[j][i][w] = v[w];
            } else {
              const u32x2_t v = *reinterpret_cast<const u32x2_t*>(p);
              vf[j][i][0] = v.x;
              vf[j][i][1] = v.y;
            }
          }
        }
      }
      f32x4_t s[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < D / 32; ++i) s[t] = at_mfma<T>(kf[t][i], qf[i], s[t]);
      }
      Pages after{0, 0};
      if (key0 + kDaStep < stop) {
        __builtin_amdgcn_sched_barrier(0);
        if (key0 + 2 * kDaStep < stop) after = pages(key0 + 2 * kDaStep);
        if (kEarly) keys(key0 + kDaStep, next.k);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (key0 < seq.first || key0 + 32 > seq.len || __any(bad)) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = key0 + 8 * c + 4 * t + i;
            // a page that the cache does not have, or a length that the table does not
            // cover: not a number, and so is the output
            s[t][i] = key < seq.first || key >= seq.len ? -INFINITY : bad ? NAN : s[t][i];
          }
      }
      // exponents from the running maximum as it is (as k_attention's, but for kTop, which
      // is added last: heads of 512 have no register for it in the branch)
      float top = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[t][i] = __builtin_fmaf(s[t][i], a.scale2, -m);
          top = fmaxf(top, s[t][i]);
        }
      if (__any(top > (l == 0.f ? -INFINITY : AtWeight<T>::kOver - AtWeight<T>::kTop))) {
        const float t = at_max_over_c(top);
        const bool first = at_sum_over_c(l) == 0.f;
        const float up = t > (first ? -INFINITY : 0.f) ? t : 0.f;
        const float f = first ? 1.f : __builtin_amdgcn_exp2f(-up);  // (0 x 2^-up need not be a number)
        m += up;
        l *= f;
        s[0] -= up;
        s[1] -= up;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int e = 0; e < VW; ++e) acc[j][e] *= f;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[t][i] = __builtin_amdgcn_exp2f(AtWeight<T>::kTop == 0.f ? s[t][i] : s[t][i] + AtWeight<T>::kTop);
          l += s[t][i];
        }
      const u32x4_t p = at_pack8<T>(s[0], s[1]);
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          // column e of the block, its eight keys in their order
          const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
          u32x4_t v;
#pragma unroll
          for (int w = 0; w < 4; ++w) v[w] = __builtin_amdgcn_perm(vf[j][2 * w + 1][e / 2], vf[j][2 * w][e / 2], sel);
          acc[j][e] = at_mfma<T>(v, p, acc[j][e]);
        }
      now = next;
      next = after;
    }

    // the wavefronts' sums, joined (a wavefront without keys has no maximum)
    l = at_sum_over_c(l);
    if (l == 0.f) m = -INFINITY;
    if (c == 0) {
      sm[wave][r] = m;
      sl[wave][r] = l;
    }
    __syncthreads();
    float top = sm[0][r];
#pragma unroll
    for (int w = 1; w < kDaWaves; ++w) top = fmaxf(top, sm[w][r]);
    if (top == -INFINITY) top = 0.f;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kDaWaves; ++w) sum += sl[w][r] * __builtin_amdgcn_exp2f(sm[w][r] - top);
    const float f = __builtin_amdgcn_exp2f(m - top);
    if (r < q_n) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int e = 0; e < VW; ++e)
          *reinterpret_cast<f32x4_t*>(so + (wave * NB + j) * VW * 256 + e * 256 + lane * 4) = acc[j][e] * f;
    }
    __syncthreads();
    const bool whole = s0 == 0 && s1 == seq.steps;
    float* part = a.part + (int64_t)(2 * blockIdx.x + (pos == begin ? 0 : 1)) * (16 * (D + 2));
    // thread: columns 16 VW j + VW (4 c + i) .. of query r
    if (r < q_n) {
      // a sum of zero: no keys, or scores of -infinity alone, whose softmax is not a number
      const float inv = sum != 0.f ? 1.0f / sum : seq.len > 0 ? NAN : 0.f;
      for (int w = wave; w < NB * 4; w += kDaWaves) {
        const int j = w >> 2, i = w & 3;
        float v[VW];
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          v[e] = 0.f;
#pragma unroll
          for (int u = 0; u < kDaWaves; ++u) v[e] += so[(u * NB + j) * VW * 256 + e * 256 + lane * 4 + i];
        }
        const int d = 16 * VW * j + VW * (4 * c + i);
        if (whole) {
          unsigned char* o = static_cast<unsigned char*>(a.out) + ((int64_t)b * a.Hq + head0 + r) * (D * 2) + 2 * d;
#pragma unroll
          for (int e = 0; e < VW; e += 4)
            *reinterpret_cast<u32x2_t*>(o + 2 * e) =
                u32x2_t{at_pack2<T>(v[e] * inv, v[e + 1] * inv), at_pack2<T>(v[e + 2] * inv, v[e + 3] * inv)};
        } else {
#pragma unroll
          for (int e = 0; e < VW; e += 4)
            *reinterpret_cast<f32x4_t*>(part + r * D + d + e) = f32x4_t{v[e], v[e + 1], v[e + 2], v[e + 3]};
        }
      }
      if (!whole && wave == 0 && c == 0) {
        part[16 * D + r] = sum == 0.f ? -INFINITY : top;  // (no maximum: it must not outweigh a lower one)
        part[16 * D + 16 + r] = sum;
      }
    }
    pos += s1 - s0;
    if (unit == units - 1 && s1 == seq.steps) {
      at += seq.steps * units;
      ++b;
    }
    __syncthreads();
  }
}

// The pieces of a query added up, in an order set by their number: a workgroup
// for each query of each (sequence, head), nothing to do where one workgroup had
// all its steps.  256 / (D / 4) groups of threads take a part of the pieces each.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_decode_join(DecodeAttnArgs a) {
  constexpr int L = D / 4, P = 256 / L;
  __shared__ __align__(16) float sv[P][D];
  __shared__ float sl[P];
  const int lane = threadIdx.x & 63;
  const int gt = (a.group + 15) / 16, units = a.Hk * gt;
  const int b = blockIdx.x / units, unit = blockIdx.x - b * units, q = blockIdx.y;
  const int hk = unit / gt, q_first = (unit - hk * gt) * 16;
  if (q_first + q >= a.group) return;
  const DaSeq seq = da_seq(a, b);
  const int total = da_before(a, a.B) * units;
  const int first = da_before(a, b) * units + unit * seq.steps, last = first + seq.steps - 1;
  const int groups = min(a.groups, total);
  // the workgroup that has a step: the last whose start is not behind it
  auto owner = [&](int step) { return (int)(((int64_t)(step + 1) * groups - 1) / total); };
  const int g0 = owner(first), g1 = owner(last);
  if (g0 == g1) return;
  // the first piece is its workgroup's second where the unit does not start with it
  const bool opens = da_start(g0, groups, total) >= first;
  auto piece = [&](int g) { return a.part + (int64_t)(2 * g + (g == g0 && !opens ? 1 : 0)) * (16 * (D + 2)); };
  float top = -INFINITY;
  for (int g = g0 + lane; g <= g1; g += 64) top = fmaxf(top, piece(g)[16 * D + q]);
  top = wave_max_f32(top);
  if (top == -INFINITY) top = 0.f;
  const int at = threadIdx.x / L, d = 4 * (threadIdx.x % L);
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll 4
  for (int g = g0 + at; g <= g1; g += P) {
    const float* p = piece(g);
    const float f = __builtin_amdgcn_exp2f(p[16 * D + q] - top);
    v += *reinterpret_cast<const f32x4_t*>(p + q * D + d) * f;
    l += p[16 * D + 16 + q] * f;
  }
  *reinterpret_cast<f32x4_t*>(&sv[at][d]) = v;
  if (d == 0) sl[at] = l;
  __syncthreads();
  if (at != 0) return;
#pragma unroll
  for (int i = 1; i < P; ++i) {
    v += *reinterpret_cast<const f32x4_t*>(&sv[i][d]);
    l += sl[i];
  }
  const float inv = l != 0.f ? 1.0f / l : seq.len > 0 ? NAN : 0.f;
  *reinterpret_cast<u32x2_t*>(static_cast<unsigned char*>(a.out) +
                              ((int64_t)b * a.Hq + hk * a.group + q_first + q) * (D * 2) + 2 * d) =
      u32x2_t{at_pack2<T>(v[0] * inv, v[1] * inv), at_pack2<T>(v[2] * inv, v[3] * inv)};
}

namespace {

template <typename T, int D>
hipError_t decode(const DecodeAttnArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((k_decode_attention<T, D>), dim3(a.groups), dim3(64 * kDaWaves), kDaWaves * D * 16 * 4, s, a);
  if (!a.whole)
    hipLaunchKernelGGL((k_decode_join<T, D>), dim3((unsigned)(a.B * a.Hk * ((a.group + 15) / 16)),
                                                    (unsigned)(a.group < 16 ? a.group : 16)),
                       dim3(256), 0, s, a);
  return hipGetLastError();
}

template <typename T>
hipError_t decode_type(const DecodeAttnArgs& a, hipStream_t s) {
  switch (a.D) {
    case 64: return decode<T, 64>(a, s);
    case 128: return decode<T, 128>(a, s);
    case 256: return decode<T, 256>(a, s);
    case 512: return decode<T, 512>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

// Few steps: a workgroup has all of a (sequence, head)'s, without pieces and their join,
// which cost about 4 us of both sides (181 keys, heads of 256: 16.7 -> 12.3 us a call;
// 4 x 1000 keys of 128 16.2 -> 14.4; too many, 1000 keys of 256 16.6 -> 25.8, 512 of 512
// 20.3 -> 29.1).  "Few" is said of the table's width, which the host knows: a short sequence
// in a wide table, or a window, is dealt out all the same (181 keys in a table for 8192: 14.0 us
// where one of three pages takes 10.1).
bool decode_attn_whole(int64_t D, int64_t keys) { return keys <= kDaStep * std::min<int64_t>(8, 1024 / D); }
int decode_attn_groups(int64_t B, int64_t Hq, int64_t Hk, int64_t D, int64_t keys) {
  if (decode_attn_whole(D, keys)) return (int)(B * Hk * ((Hq / Hk + 15) / 16));
  const int64_t steps = (keys + kDaStep - 1) / kDaStep + 1;  // a window may start inside one
  const int64_t units = B * Hk * ((Hq / Hk + 15) / 16);
  return units * steps < kDecodeAttnGroups ? (int)(units * steps) : kDecodeAttnGroups;
}
size_t decode_attn_part_floats(int64_t groups, int64_t D) { return (size_t)groups * 2 * 16 * (D + 2); }

hipError_t launch_decode_attention(int dtype, const DecodeAttnArgs& a, hipStream_t s) {
  return dtype == 0 ? decode_type<__bf16>(a, s) : decode_type<_Float16>(a, s);
}

}  // namespace w4a16
