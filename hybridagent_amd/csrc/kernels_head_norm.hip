// RMS norm of every head of queries, keys and values with the position rotation
// in the same pass, its gradients, and the form that writes keys and values into
// a paged cache (include/w4a16moe.h: w4a16_head_norm_rope, .._backward,
// w4a16_append_kv).  A row is a head of a token, D elements:
//
//   r = rsqrt(mean x^2 + eps), u = x r w
//   y_i = u_i cos_i - u_{i+h} sin_i, y_{i+h} = u_{i+h} cos_i + u_i sin_i   (i < h = R / 2)
//
// backward, with g = dy turned back by the same angles and t = g w:
//   dx = r (t - x r mean(t x r)),  dw = sum over rows of g x r
//
// Bound: memory (one read and one write of each row; 8191 tokens of 32 heads of 256:
// forward 58 us, 4.6 TB/s, where a copy reaches 4.95; backward 91 us, two reads and a
// write, 4.4, and 8 for the join of the weights' partial rows; fp32, twice the bytes,
// 102 and 181 with the join; into the cache 4097 tokens of 16 + 2 + 2 heads of 512 35 us,
// 4.8, and 2 more with dense keys and values for the prompt).  L lanes have a row, each
// two pieces of four elements: of the turned columns piece i and its partner R / 2
// further, of the others neighbours, so that a pair never leaves its lane and an
// angle is read once.  A wavefront takes kHnRows groups of 64 / L rows of one
// token, loaded together, and its token's angles once for them.
#include <type_traits>

#include "attention.hpp"

namespace w4a16 {

namespace {

constexpr int kHnRows = 4;
constexpr int kHnBackBlocks = 1024;

// the number of lanes of a row
inline int hn_lanes(int64_t D) { return D <= 64 ? 8 : D <= 128 ? 16 : D <= 256 ? 32 : 64; }
inline int64_t hn_tasks(int64_t T, int64_t heads, int64_t D) {
  const int per = kHnRows * (64 / hn_lanes(D));
  return T * ((heads + per - 1) / per);
}

// a lane's elements of a row: pieces at a and b
struct HnPlace {
  int a, b;
  bool in, turned;
};
__device__ __forceinline__ HnPlace hn_place(const HeadNormArgs& g, int j) {
  HnPlace p;
  p.turned = 8 * j < g.R;
  p.a = p.turned ? 4 * j : 8 * j;
  p.b = p.turned ? 4 * j + (g.R >> 1) : 8 * j + 4;
  p.in = 8 * j < g.D;
  return p;
}
template <typename T>
struct Hn8 {
  static constexpr int kWords = sizeof(T);  // of a piece
  typedef __attribute__((ext_vector_type(kWords))) uint32_t piece_t;
  piece_t w[2];
  __device__ __forceinline__ void load(const void* row, const HnPlace& p) {
    w[0] = *reinterpret_cast<const piece_t*>(static_cast<const T*>(row) + p.a);
    w[1] = *reinterpret_cast<const piece_t*>(static_cast<const T*>(row) + p.b);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[0][i] = w[1][i] = 0;
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4)
      return __uint_as_float(w[i >> 2][i & 3]);
    else
      return i & 1 ? at_hi<T>(w[i >> 2][(i & 3) >> 1]) : at_lo<T>(w[i >> 2][(i & 3) >> 1]);
  }
};
template <typename T>
__device__ __forceinline__ void hn_store(void* row, const HnPlace& p, const float (&v)[8]) {
  typedef typename Hn8<T>::piece_t piece_t;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float* x = v + 4 * h;
    piece_t w;
    if constexpr (sizeof(T) == 4)
      w = piece_t{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
    else
      w = piece_t{at_pack2<T>(x[0], x[1]), at_pack2<T>(x[2], x[3])};
    *reinterpret_cast<piece_t*>(static_cast<T*>(row) + (h ? p.b : p.a)) = w;
  }
}

// a lane's angles; not turned: cos 1, sin 0
struct HnTurn {
  f32x4_t cos, sin;
};
// dir: 1, or -1 to turn back.  A position that the tables do not have: not a number.
__device__ __forceinline__ HnTurn hn_turn(const HeadNormArgs& g, int t, const HnPlace& p, float dir) {
  const int pos = g.pos[t];
  const bool bad = pos < 0 || pos >= g.P;
  HnTurn n;
  n.cos = f32x4_t{1.f, 1.f, 1.f, 1.f};
  n.sin = f32x4_t{0.f, 0.f, 0.f, 0.f};
  if (p.turned && !bad) {
    const int64_t at = (int64_t)pos * (g.R >> 1) + p.a;
    n.cos = *reinterpret_cast<const f32x4_t*>(g.cos + at);
    n.sin = *reinterpret_cast<const f32x4_t*>(g.sin + at) * dir;
  }
  if (bad) n.cos = n.sin = f32x4_t{NAN, NAN, NAN, NAN};
  return n;
}
// (Columns that are not turned are neighbours in u, not a pair: with a sine of zero one that is
// not finite would make a finite one not a number.)
__device__ __forceinline__ void hn_rotate(const HnTurn& n, bool turned, float (&u)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = u[i], y = u[4 + i];
    u[i] = x * n.cos[i] - (turned ? y : 0.f) * n.sin[i];
    u[4 + i] = y * n.cos[i] + (turned ? x : 0.f) * n.sin[i];
  }
}

// head h of token t: its row in the inputs, what it is (0: query, 1: key, 2:
// value) and its number among these
struct HnRow {
  int kind, head;
  const unsigned char* x;
};
__device__ __forceinline__ HnRow hn_row(const HeadNormArgs& a, int t, int h) {
  HnRow r;
  r.kind = h < a.Hq ? 0 : h < a.Hq + a.Hk ? 1 : 2;
  r.head = h - (r.kind == 0 ? 0 : r.kind == 1 ? a.Hq : a.Hq + a.Hk);
  const void* p = r.kind == 0 ? a.q : r.kind == 1 ? a.k : a.v;
  const int64_t tok = r.kind == 0 ? a.q_tok : r.kind == 1 ? a.k_tok : a.v_tok;
  const int64_t one = r.kind == 0 ? a.q_head : r.kind == 1 ? a.k_head : a.v_head;
  r.x = static_cast<const unsigned char*>(p) + t * tok + r.head * one;
  return r;
}

}  // namespace

template <typename T, int L, bool PAGED>
__global__ __launch_bounds__(256) void k_head_norm(HeadNormArgs a, int chunks) {
  constexpr int RP = 64 / L;
  const int lane = threadIdx.x & 63, j = lane % L, sub = lane / L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t task = (int64_t)blockIdx.x * 4 + wave;
  const int t = (int)(task / chunks);
  if (t >= a.T) return;
  const int heads = a.Hq + a.Hk + (a.v != nullptr ? a.Hk : 0);
  const int h0 = (int)(task - (int64_t)t * chunks) * (kHnRows * RP) + sub;
  const HnPlace at = hn_place(a, j);

  HnRow row[kHnRows];
  Hn8<T> x[kHnRows];
#pragma unroll
  for (int i = 0; i < kHnRows; ++i) {
    const int h = h0 + RP * i;
    row[i] = hn_row(a, t, min(h, heads - 1));
    if (at.in && h < heads)
      x[i].load(row[i].x, at);
    else
      x[i].zero();
  }
  const HnTurn turn = hn_turn(a, t, at, 1.f);
  const int slot = PAGED ? a.slots[t] : 0;
  const int page = PAGED ? slot / a.page : 0;
  const bool kept = PAGED ? slot >= 0 && slot < a.slots_n : true;
#pragma unroll
  for (int i = 0; i < kHnRows; ++i) {
    const int h = h0 + RP * i, kind = row[i].kind;
    const void* w = kind == 0 ? a.qw : kind == 1 ? a.kw : nullptr;
    float u[8], sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      u[e] = x[i].get(e);
      sum = __builtin_fmaf(u[e], u[e], sum);
    }
    sum = at_sum_over<L>(sum);
    const bool norm = kind == 2 ? a.v_norm : w != nullptr;
    const float f = norm ? __frsqrt_rn(sum / (float)a.D + a.eps) : 1.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] *= f;
    if (w != nullptr && at.in) {
      Hn8<T> wv;
      wv.load(w, at);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] *= wv.get(e);
    }
    if (kind != 2) hn_rotate(turn, at.turned, u);
    if (!at.in || h >= heads) continue;
    const int n = row[i].head;
    void* o = kind == 0 ? a.yq : kind == 1 ? a.yk : a.yv;
    if (!PAGED || o != nullptr)
      hn_store<T>(static_cast<T*>(o) + ((int64_t)t * (kind == 0 ? a.Hq : a.Hk) + n) * a.D, at, u);
    if (PAGED && kept && kind != 0) {
      unsigned char* to =
          static_cast<unsigned char*>(kind == 1 ? a.kc : a.vc) + page * (kind == 1 ? a.k_page : a.v_page);
      hn_store<T>(to + ((int64_t)n * a.page + (slot - page * a.page)) * a.D * sizeof(T), at, u);
    }
  }
}

template <typename T, int L>
__global__ __launch_bounds__(256) void k_head_norm_backward(HeadNormArgs a, int chunks, int64_t tasks) {
  constexpr int RP = 64 / L;
  const int lane = threadIdx.x & 63, j = lane % L, sub = lane / L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = a.Hq + a.Hk + (a.v != nullptr ? a.Hk : 0);
  const HnPlace at = hn_place(a, j);
  const float over = 1.0f / (float)a.D;
  float dw[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[0][e] = dw[1][e] = 0.f;
  Hn8<T> wq, wk;
  wq.zero();
  wk.zero();
  if (a.qw != nullptr && at.in) {
    wq.load(a.qw, at);
    wk.load(a.kw, at);
  }

  for (int64_t task = (int64_t)blockIdx.x * 4 + wave; task < tasks; task += (int64_t)gridDim.x * 4) {
    const int t = (int)(task / chunks);
    const int h0 = (int)(task - (int64_t)t * chunks) * (kHnRows * RP) + sub;
    Hn8<T> x[kHnRows], dy[kHnRows];
#pragma unroll
    for (int i = 0; i < kHnRows; ++i) {
      const int h = h0 + RP * i;
      const HnRow row = hn_row(a, t, min(h, heads - 1));
      const void* d = row.kind == 0 ? a.dq : row.kind == 1 ? a.dk : a.dv;
      if (at.in && h < heads) {
        x[i].load(row.x, at);
        dy[i].load(static_cast<const T*>(d) + ((int64_t)t * (row.kind == 0 ? a.Hq : a.Hk) + row.head) * a.D, at);
      } else {
        x[i].zero();
        dy[i].zero();
      }
    }
    const HnTurn turn = hn_turn(a, t, at, -1.f);
#pragma unroll
    for (int i = 0; i < kHnRows; ++i) {
      const int h = h0 + RP * i;
      const HnRow row = hn_row(a, t, min(h, heads - 1));
      const int kind = row.kind;
      const bool norm = kind == 2 || a.qw != nullptr;
      float g[8], xh[8], sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xh[e] = x[i].get(e);
        sum = __builtin_fmaf(xh[e], xh[e], sum);
        g[e] = dy[i].get(e);
      }
      const float f = __frsqrt_rn(at_sum_over<L>(sum) * over + a.eps);
      if (kind != 2) hn_rotate(turn, at.turned, g);
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xh[e] *= f;
        if (h < heads && at.in) {
          dw[0][e] += kind == 0 ? g[e] * xh[e] : 0.f;
          dw[1][e] += kind == 1 ? g[e] * xh[e] : 0.f;
        }
        if (norm && kind != 2) g[e] *= kind == 0 ? wq.get(e) : wk.get(e);
        dot = __builtin_fmaf(g[e], xh[e], dot);
      }
      dot = at_sum_over<L>(dot) * over;
      if (norm) {
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = f * (g[e] - xh[e] * dot);
      }
      if (!at.in || h >= heads) continue;
      void* o = kind == 0 ? a.yq : kind == 1 ? a.yk : a.yv;
      hn_store<T>(static_cast<T*>(o) + ((int64_t)t * (kind == 0 ? a.Hq : a.Hk) + row.head) * a.D, at, g);
    }
  }
  if (a.part == nullptr) return;
  // over the wavefront's rows, then over the wavefronts
  __shared__ float all[4][2][kHeadNormMaxD];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v = dw[k][e];
#pragma unroll
      for (int o = L; o < 64; o <<= 1) v += __shfl_xor(v, o);
      if (sub == 0 && at.in) all[wave][k][(e < 4 ? at.a : at.b - 4) + e] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.D; i += 256) {
    const int k = i >= a.D, d = i - k * a.D;
    a.part[(int64_t)blockIdx.x * 2 * a.D + i] = (all[0][k][d] + all[1][k][d]) + (all[2][k][d] + all[3][k][d]);
  }
}

namespace {

template <typename T, bool PAGED>
hipError_t head_norm(const HeadNormArgs& a, hipStream_t s) {
  const int heads = a.Hq + a.Hk + (a.v != nullptr ? a.Hk : 0), L = hn_lanes(a.D), per = kHnRows * (64 / L);
  const int chunks = (heads + per - 1) / per;
  const dim3 grid((unsigned)(((int64_t)a.T * chunks + 3) / 4));
  switch (L) {
    case 8: hipLaunchKernelGGL((k_head_norm<T, 8, PAGED>), grid, dim3(256), 0, s, a, chunks); break;
    case 16: hipLaunchKernelGGL((k_head_norm<T, 16, PAGED>), grid, dim3(256), 0, s, a, chunks); break;
    case 32: hipLaunchKernelGGL((k_head_norm<T, 32, PAGED>), grid, dim3(256), 0, s, a, chunks); break;
    case 64: hipLaunchKernelGGL((k_head_norm<T, 64, PAGED>), grid, dim3(256), 0, s, a, chunks); break;
  }
  return hipGetLastError();
}

template <typename T>
hipError_t head_norm_back(const HeadNormArgs& a, hipStream_t s) {
  const int heads = a.Hq + a.Hk + (a.v != nullptr ? a.Hk : 0), L = hn_lanes(a.D), per = kHnRows * (64 / L);
  const int chunks = (heads + per - 1) / per;
  const int64_t tasks = (int64_t)a.T * chunks;
  const dim3 grid((unsigned)head_norm_partials(a.T, heads, a.D));
  switch (L) {
    case 8: hipLaunchKernelGGL((k_head_norm_backward<T, 8>), grid, dim3(256), 0, s, a, chunks, tasks); break;
    case 16: hipLaunchKernelGGL((k_head_norm_backward<T, 16>), grid, dim3(256), 0, s, a, chunks, tasks); break;
    case 32: hipLaunchKernelGGL((k_head_norm_backward<T, 32>), grid, dim3(256), 0, s, a, chunks, tasks); break;
    case 64: hipLaunchKernelGGL((k_head_norm_backward<T, 64>), grid, dim3(256), 0, s, a, chunks, tasks); break;
  }
  return hipGetLastError();
}

}  // namespace

int head_norm_partials(int64_t T, int64_t heads, int64_t D) {
  const int64_t blocks = (hn_tasks(T, heads, D) + 3) / 4;
  return (int)(blocks < kHnBackBlocks ? blocks : kHnBackBlocks);
}

hipError_t launch_head_norm(int dtype, bool paged, const HeadNormArgs& a, hipStream_t s) {
  if (paged) return dtype == 0 ? head_norm<__bf16, true>(a, s) : head_norm<_Float16, true>(a, s);
  switch (dtype) {
    case 0: return head_norm<__bf16, false>(a, s);
    case 1: return head_norm<_Float16, false>(a, s);
    default: return head_norm<float, false>(a, s);
  }
}

hipError_t launch_head_norm_backward(int dtype, const HeadNormArgs& a, hipStream_t s) {
  switch (dtype) {
    case 0: return head_norm_back<__bf16>(a, s);
    case 1: return head_norm_back<_Float16>(a, s);
    default: return head_norm_back<float>(a, s);
  }
}

}  // namespace w4a16
