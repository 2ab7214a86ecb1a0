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
// Bound: memory (one read and one write of each row).  L lanes have a row, 8
// elements each, so that every load is 16 bytes a lane and whole lines; a
// wavefront takes kHnRows groups of 64 / L rows of one token, loaded together,
// and reads its token's angles once for them.  The two halves of a rotated pair
// meet through the wavefront's own LDS rows.
#include <type_traits>

#include "attention.hpp"

namespace w4a16 {

namespace {

constexpr int kHnRows = 4;
constexpr int kHnBackBlocks = 512;

// the number of lanes of a row
inline int hn_lanes(int64_t D) { return D <= 64 ? 8 : D <= 128 ? 16 : D <= 256 ? 32 : 64; }
inline int64_t hn_tasks(int64_t T, int64_t heads, int64_t D) {
  const int per = kHnRows * (64 / hn_lanes(D));
  return T * ((heads + per - 1) / per);
}

// eight elements
template <typename T>
struct Hn8 {
  static constexpr int kWords = 2 * sizeof(T);
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const void* p) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      const u32x4_t v = ld16(static_cast<const uint32_t*>(p) + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[i + j] = v[j];
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4)
      return __uint_as_float(w[i]);
    else
      return i & 1 ? at_hi<T>(w[i / 2]) : at_lo<T>(w[i / 2]);
  }
};
template <typename T>
__device__ __forceinline__ void hn_store(void* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    st16(p, u32x4_t{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
    st16(static_cast<char*>(p) + 16,
         u32x4_t{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])});
  } else {
    st16(p, u32x4_t{at_pack2<T>(v[0], v[1]), at_pack2<T>(v[2], v[3]), at_pack2<T>(v[4], v[5]), at_pack2<T>(v[6], v[7])});
  }
}

template <int L>
__device__ __forceinline__ float hn_sum(float v) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

// A lane's angles for elements 8 j .. 8 j + 7 of a rotated row, in two groups of
// four: y = cos u + sin u', u' the element `to` further (sin with its sign)
struct HnTurn {
  float cos[8], sin[8];
  int to[2];
};
// dir: 1, or -1 to turn back.  h = R / 2, a multiple of four.
__device__ __forceinline__ HnTurn hn_turn(const HeadNormArgs& a, int t, int j, float dir) {
  HnTurn n;
  const int h = a.R >> 1, p = a.pos[t];
  const bool bad = p < 0 || p >= a.P;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int e = 8 * j + 4 * g;
    const bool low = e < h, turned = e < a.R;
    n.to[g] = low && turned ? h : turned ? -h : 0;
    f32x4_t c = {1.f, 1.f, 1.f, 1.f}, s = {0.f, 0.f, 0.f, 0.f};
    if (turned && !bad) {
      const int64_t at = (int64_t)p * h + (low ? e : e - h);
      c = *reinterpret_cast<const f32x4_t*>(a.cos + at);
      s = *reinterpret_cast<const f32x4_t*>(a.sin + at) * (low ? -dir : dir);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // a position that the tables do not have: not a number
      n.cos[4 * g + i] = bad ? NAN : c[i];
      n.sin[4 * g + i] = s[i];
    }
  }
  return n;
}
// u turned, through the row's LDS place (of this wavefront alone)
__device__ __forceinline__ void hn_rotate(const HnTurn& n, float* row, int j, float (&u)[8]) {
  float* p = row + 8 * j;
#pragma unroll
  for (int g = 0; g < 2; ++g)
    *reinterpret_cast<f32x4_t*>(p + 4 * g) = f32x4_t{u[4 * g], u[4 * g + 1], u[4 * g + 2], u[4 * g + 3]};
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const f32x4_t v = *reinterpret_cast<const f32x4_t*>(p + 4 * g + n.to[g]);
#pragma unroll
    for (int i = 0; i < 4; ++i) u[4 * g + i] = u[4 * g + i] * n.cos[4 * g + i] + v[i] * n.sin[4 * g + i];
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
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
  __shared__ __align__(16) float rows[4][64 * 8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane % L, sub = lane / L;
  const int64_t task = (int64_t)blockIdx.x * 4 + wave;
  const int t = (int)(task / chunks);
  if (t >= a.T) return;
  const int heads = a.Hq + a.Hk + (a.v != nullptr ? a.Hk : 0);
  const int h0 = (int)(task - (int64_t)t * chunks) * (kHnRows * RP) + sub;
  const bool in = 8 * j < a.D;

  HnRow row[kHnRows];
  Hn8<T> x[kHnRows];
#pragma unroll
  for (int i = 0; i < kHnRows; ++i) {
    const int h = h0 + RP * i;
    row[i] = hn_row(a, t, min(h, heads - 1));
    if (in && h < heads)
      x[i].load(row[i].x + 8 * j * sizeof(T));
    else
      x[i].zero();
  }
  const HnTurn turn = hn_turn(a, t, j, 1.f);
  const int slot = PAGED ? a.slots[t] : 0;
  const int page = PAGED ? slot / a.page : 0;
  const bool kept = PAGED ? slot >= 0 && slot < a.slots_n : true;
  float* place = rows[wave] + sub * (L * 8);
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
    sum = hn_sum<L>(sum);
    const bool norm = kind == 2 ? a.v_norm : w != nullptr;
    const float f = norm ? __frsqrt_rn(sum / (float)a.D + a.eps) : 1.f;
    Hn8<T> wv;
    if (w != nullptr && in) wv.load(static_cast<const unsigned char*>(w) + 8 * j * sizeof(T));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      u[e] *= f;
      if (w != nullptr && in) u[e] *= wv.get(e);
    }
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = u[e];
    hn_rotate(turn, place, j, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = kind == 2 ? u[e] : y[e];
    if (!in || h >= heads) continue;
    const int n = row[i].head;
    if (!PAGED || kind == 0) {
      void* o = kind == 0 ? a.yq : kind == 1 ? a.yk : a.yv;
      hn_store<T>(static_cast<T*>(o) + ((int64_t)t * (kind == 0 ? a.Hq : a.Hk) + n) * a.D + 8 * j, y);
    } else if (kept) {
      unsigned char* o = static_cast<unsigned char*>(kind == 1 ? a.yk : a.yv) + page * (kind == 1 ? a.k_page : a.v_page);
      hn_store<T>(o + (((int64_t)n * a.page + (slot - page * a.page)) * a.D + 8 * j) * sizeof(T), y);
    }
  }
}

template <typename T, int L>
__global__ __launch_bounds__(256) void k_head_norm_backward(HeadNormArgs a, int chunks, int64_t tasks) {
  constexpr int RP = 64 / L;
  __shared__ __align__(16) float rows[4][64 * 8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane % L, sub = lane / L;
  const int heads = a.Hq + a.Hk + (a.v != nullptr ? a.Hk : 0);
  const bool in = 8 * j < a.D;
  const float over = 1.0f / (float)a.D;
  float* place = rows[wave] + sub * (L * 8);
  float dw[2][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) dw[0][e] = dw[1][e] = 0.f;
  Hn8<T> wq, wk;
  wq.zero();
  wk.zero();
  if (a.qw != nullptr && in) {
    wq.load(static_cast<const T*>(a.qw) + 8 * j);
    wk.load(static_cast<const T*>(a.kw) + 8 * j);
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
      const int64_t at = ((int64_t)t * (row.kind == 0 ? a.Hq : a.Hk) + row.head) * a.D + 8 * j;
      if (in && h < heads) {
        x[i].load(row.x + 8 * j * sizeof(T));
        dy[i].load(static_cast<const T*>(d) + at);
      } else {
        x[i].zero();
        dy[i].zero();
      }
    }
    const HnTurn turn = hn_turn(a, t, j, -1.f);
#pragma unroll
    for (int i = 0; i < kHnRows; ++i) {
      const int h = h0 + RP * i;
      const HnRow row = hn_row(a, t, min(h, heads - 1));
      const int kind = row.kind;
      const bool norm = kind == 2 || a.qw != nullptr;
      float g[8], u[8], sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = x[i].get(e);
        sum = __builtin_fmaf(v, v, sum);
        u[e] = g[e] = dy[i].get(e);
      }
      sum = hn_sum<L>(sum);
      hn_rotate(turn, place, j, u);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = kind == 2 ? g[e] : u[e];
      const float f = __frsqrt_rn(sum * over + a.eps);
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xh = x[i].get(e) * f;
        if (h < heads && in) {
          dw[0][e] += kind == 0 ? g[e] * xh : 0.f;
          dw[1][e] += kind == 1 ? g[e] * xh : 0.f;
        }
        u[e] = kind == 2 ? g[e] : g[e] * (kind == 0 ? wq.get(e) : wk.get(e));
        dot = __builtin_fmaf(u[e], xh, dot);
      }
      dot = hn_sum<L>(dot) * over;
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = norm ? f * (u[e] - x[i].get(e) * f * dot) : g[e];
      if (!in || h >= heads) continue;
      void* o = kind == 0 ? a.yq : kind == 1 ? a.yk : a.yv;
      hn_store<T>(static_cast<T*>(o) + ((int64_t)t * (kind == 0 ? a.Hq : a.Hk) + row.head) * a.D + 8 * j, u);
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
      if (sub == 0) all[wave][k][8 * j + e] = v;
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
