// Layer norm and its backward pass for rows of bf16, fp16 or fp32 (weights in
// the rows' type, everything computed in fp32), and for HybridLink's bf16 rows
// beside fp32 ones (LnForm):
//   mean = sum x / H, rstd = 1 / sqrt(sum (x - mean)^2 / H + eps)
//   y = (x - mean) rstd w + b
//   xh = (x - mean) rstd, g = dy w
//   dx = rstd (g - sum g / H - xh sum(g xh) / H) (+ add)
//   dw = sum over rows of dy xh, db = sum over rows of dy
// The variance is of the deviations from the mean (a second pass over the row
// in registers), not a difference of squares.
//
// A row is held in registers by TPR threads, EPT elements each: a wavefront
// (no LDS, no barrier) or a workgroup.  Loads are 16 bytes per lane where
// rows and pointers allow it (VEC elements), else one element.  The weights
// are loaded once per thread and kept across its rows.
//
// Bound: forward HBM: 8192 bf16 rows of 2816 15.7 us (5.9 TB/s, part of it from
// the 256 MB cache); one row 2.4.  Backward, the same rows: 2049 13.2 us, 4099
// 18.1 and the join 4.0: a further row comes at the memory's rate, some 9 us do
// not depend on the rows (the first one's latency, the join of a workgroup's
// wavefronts, the partial rows).  The column sums of the backward pass are kept in registers
// across the rows of a thread, added over a workgroup's wavefronts in LDS and
// written once per workgroup (kLnPartials at most); a second launch
// (k_column_join) adds those in order, so that a repeated call gives the same
// bits (another alignment of the pointers takes other loads and another order).
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"

namespace w4a16 {

namespace {

template <typename T>
struct LnType;
template <>
struct LnType<__bf16> {
  static __device__ __forceinline__ float load(uint32_t bits) { return bf16_bits_to_f32(bits); }
};
template <>
struct LnType<_Float16> {
  static __device__ __forceinline__ float load(uint32_t bits) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
  }
};

// a thread's EPT elements of a row as they lie in memory: chunk q of thread t
// of TPR is elements (t + TPR q) VEC ..; those past the row read as zero and
// are not stored (the row's buffer descriptor ends with it)
template <typename T, int VEC, int EPT, int TPR>
struct LnRaw {
  static constexpr int NQ = EPT / VEC;
  static constexpr int kChunk = VEC * (int)sizeof(T);
  static constexpr int kWords = kChunk / 4 > 0 ? kChunk / 4 : 1;
  uint32_t w[NQ][kWords];

  __device__ __forceinline__ void load(const void* row, int t, int H) {
    const auto r = make_rsrc(row, (uint32_t)(H * (int)sizeof(T)));
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int o = t * kChunk + TPR * q * kChunk;
      if constexpr (VEC > 1) {
        load_chunk(r, q, o);
      } else if constexpr (sizeof(T) == 4) {
        w[q][0] = __builtin_amdgcn_raw_buffer_load_b32(r, o, 0, 0);
      } else {
        w[q][0] = buf_ld_u16(r, o);
      }
    }
  }
  // VEC elements of 16 bytes, or of 32 beside 16-bit ones of 16
  __device__ __forceinline__ void load_chunk(__amdgpu_buffer_rsrc_t r, int q, int o) {
#pragma unroll
    for (int i = 0; i + 4 <= kWords; i += 4) {
      const u32x4_t v = buf_ld16(r, o, 4 * i);
      w[q][i] = v.x;
      w[q][i + 1] = v.y;
      w[q][i + 2] = v.z;
      w[q][i + 3] = v.w;
    }
  }
  __device__ __forceinline__ float get(int q, int e) const {
    if constexpr (sizeof(T) == 4)
      return __uint_as_float(w[q][e]);
    else
      return LnType<T>::load((e & 1) ? w[q][e >> 1] >> 16 : w[q][e >> 1] & 0xFFFFu);
  }
  // what is computed from the values is computed again after this, not kept
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[q][i] = opaque(w[q][i]);
  }
};

// chunk q of a row from VEC values, rounded to T
template <typename T, int VEC, int TPR>
__device__ __forceinline__ void ln_store(__amdgpu_buffer_rsrc_t r, int t, int q, const float* v) {
  constexpr int kChunk = VEC * (int)sizeof(T);
  const int o = t * kChunk + TPR * q * kChunk;
  if constexpr (VEC > 1) {
    constexpr int N = 16 / (int)sizeof(T);
    typedef T vec_t __attribute__((ext_vector_type(N)));
#pragma unroll
    for (int j = 0; j < VEC; j += N) {
      vec_t u;
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = (T)v[j + i];
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, u), r, o + j * (int)sizeof(T), 0, 0);
    }
  } else if constexpr (sizeof(T) == 4) {
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v[0]), r, o, 0, 0);
  } else {
    __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (T)v[0]), r, o, 0, 0);
  }
}

// sums of N values over the TPR threads of a row, in a fixed order
template <int TPR, int N>
__device__ __forceinline__ void ln_sum(float (&v)[N], float* part) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum_f32(v[i]);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    const int w = threadIdx.x >> 6;
    __syncthreads();  // the last sums have been read
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) part[i * W + w] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = part[i * W];
#pragma unroll
      for (int j = 1; j < W; ++j) t += part[i * W + j];
      v[i] = t;
    }
  }
}

constexpr int kLnThreads = 256;
// backward: a wavefront's rows in workgroups of eight of them
constexpr int ln_back_threads(int tpr) { return tpr > 64 ? tpr : 512; }
// the thread's row of the workgroup's (wavefront-uniform)
template <int TPR>
__device__ __forceinline__ int ln_row_of() {
  return TPR > 64 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
}

}  // namespace

template <typename T, int VEC, int EPT, int TPR, int FORM>
__global__ __launch_bounds__(kLnThreads) void k_ln_forward(LnArgs a) {
  using Raw = LnRaw<T, VEC, EPT, TPR>;
  using TX = std::conditional_t<FORM == kLnPost, float, T>;
  __shared__ float part[TPR > 64 ? TPR / 64 : 1];
  constexpr int RPB = kLnThreads / TPR;  // rows per workgroup
  const int t = threadIdx.x % TPR;
  const int H = a.H, nchunks = H / VEC;
  const float fh = (float)H;
  int64_t row = (int64_t)blockIdx.x * RPB + ln_row_of<TPR>();
  if (row >= a.M) return;  // (a workgroup per row: all of it)
  LnRaw<TX, VEC, EPT, TPR> x;
  Raw w, b;
  // the row first: its statistics wait for nothing else
  x.load(static_cast<const TX*>(a.x) + row * H, t, H);
  w.load(a.w, t, H);
  b.load(a.b != nullptr ? a.b : a.w, t, a.b != nullptr ? H : 0);
  for (;;) {
    float s[1] = {0.f};
#pragma unroll
    for (int q = 0; q < Raw::NQ; ++q)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[0] += x.get(q, e);
    ln_sum<TPR>(s, part);
    const float mean = s[0] / fh;
    float d2[1] = {0.f};
    x.forget();
#pragma unroll
    for (int q = 0; q < Raw::NQ; ++q) {
      const bool in = t + TPR * q < nchunks;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = in ? x.get(q, e) - mean : 0.f;
        d2[0] = __builtin_fmaf(d, d, d2[0]);
      }
    }
    ln_sum<TPR>(d2, part);
    const float rstd = 1.0f / sqrtf(d2[0] / fh + a.eps);
    x.forget();
    const auto yr = make_rsrc(static_cast<T*>(a.y) + row * H, (uint32_t)(H * (int)sizeof(T)));
#pragma unroll
    for (int q = 0; q < Raw::NQ; ++q) {
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = __builtin_fmaf((x.get(q, e) - mean) * rstd, w.get(q, e), b.get(q, e));
      ln_store<T, VEC, TPR>(yr, t, q, o);
    }
    if (a.mean != nullptr && t == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    row += (int64_t)gridDim.x * RPB;
    if (row >= a.M) break;
    x.load(static_cast<const TX*>(a.x) + row * H, t, H);
    w.forget();
    b.forget();
  }
}

template <typename T, int VEC, int EPT, int TPR, int FORM>
__global__ __launch_bounds__(ln_back_threads(TPR)) void k_ln_backward(LnArgs a) {
  using Raw = LnRaw<T, VEC, EPT, TPR>;
  using TX = std::conditional_t<FORM == kLnPost, float, T>;
  using TDY = std::conditional_t<FORM == kLnPre, float, T>;
  using RawF = LnRaw<float, VEC, EPT, TPR>;
  constexpr bool ADD = FORM == kLnPre;
  constexpr bool kEarly = EPT <= 32;  // registers for all of a row's `add` at once
  constexpr int RPB = ln_back_threads(TPR) / TPR;
  extern __shared__ __align__(16) float smem[];  // TPR > 64: a row's sums; else column sums, [4][2][EPT][64]
  const int t = threadIdx.x % TPR;
  const int H = a.H, nchunks = H / VEC;
  const float fh = (float)H;
  Raw w;
  w.load(a.w, t, H);
  float dw[EPT], db[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i) dw[i] = db[i] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * RPB + ln_row_of<TPR>(); row < a.M; row += (int64_t)gridDim.x * RPB) {
    LnRaw<TX, VEC, EPT, TPR> x;
    LnRaw<TDY, VEC, EPT, TPR> dy;
    RawF add;
    x.load(static_cast<const TX*>(a.x) + row * H, t, H);
    dy.load(static_cast<const TDY*>(a.dy) + row * H, t, H);
    if (ADD && kEarly) add.load(a.add + row * H, t, H);
    w.forget();
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s[2] = {0.f, 0.f};  // sum g, sum g xh
#pragma unroll
    for (int q = 0; q < Raw::NQ; ++q) {
      // past the row dy and x are zero; xh too, where -mean rstd may overflow
      const float r = t + TPR * q < nchunks ? rstd : 0.f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float xh = (x.get(q, e) - mean) * r, d = dy.get(q, e), g = d * w.get(q, e);
        s[0] += g;
        s[1] = __builtin_fmaf(g, xh, s[1]);
        dw[q * VEC + e] = __builtin_fmaf(d, xh, dw[q * VEC + e]);
        db[q * VEC + e] += d;
      }
    }
    ln_sum<TPR>(s, smem);
    const float m0 = s[0] / fh, m1 = s[1] / fh;
    x.forget();
    dy.forget();
    w.forget();
    const auto dxr = make_rsrc(static_cast<T*>(a.y) + row * H, (uint32_t)(H * (int)sizeof(T)));
    const auto dx32 = make_rsrc(a.y32 + row * H, FORM == kLnPost ? (uint32_t)H * 4u : 0u);
    const auto addr = make_rsrc(a.add + row * H, ADD ? (uint32_t)H * 4u : 0u);
#pragma unroll
    for (int q = 0; q < Raw::NQ; ++q) {
      if (ADD && !kEarly) add.load_chunk(addr, q, (t + TPR * q) * RawF::kChunk);
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float xh = (x.get(q, e) - mean) * rstd, g = dy.get(q, e) * w.get(q, e);
        o[e] = rstd * (g - m0 - xh * m1);
        if (ADD) o[e] += add.get(q, e);
      }
      ln_store<T, VEC, TPR>(dxr, t, q, o);
      if (FORM == kLnPost) ln_store<float, VEC, TPR>(dx32, t, q, o);
    }
  }
  // the wavefronts' column sums: the upper half hand theirs to the lower half,
  // until the first has them all (16 bytes per lane, a KiB per instruction)
  if constexpr (TPR == 64) {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int half = RPB / 2; half >= 1; half /= 2) {
      f32x4_t* mine = reinterpret_cast<f32x4_t*>(smem) + (wave & (half - 1)) * (EPT / 2) * 64 + t;
      if (wave >= half && wave < 2 * half) {
#pragma unroll
        for (int i = 0; i < EPT; i += 4) {
          mine[16 * i] = f32x4_t{dw[i], dw[i + 1], dw[i + 2], dw[i + 3]};
          mine[16 * (EPT + i)] = f32x4_t{db[i], db[i + 1], db[i + 2], db[i + 3]};
        }
      }
      __syncthreads();
      if (wave < half) {
#pragma unroll
        for (int i = 0; i < EPT; i += 4) {
          const f32x4_t u = mine[16 * i], v = mine[16 * (EPT + i)];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            dw[i + k] += u[k];
            db[i + k] += v[k];
          }
        }
      }
      __syncthreads();
    }
    if (wave != 0) return;
  }
  // the workgroup's, [2][H]
  const auto wr = make_rsrc(a.part + (int64_t)blockIdx.x * 2 * H, (uint32_t)(H * 4));
  const auto br = make_rsrc(a.part + (int64_t)blockIdx.x * 2 * H + H, (uint32_t)(H * 4));
#pragma unroll
  for (int q = 0; q < Raw::NQ; ++q)
#pragma unroll
    for (int e = 0; e < VEC; e += VEC < 4 ? 1 : 4) {
      const int o = ((t + TPR * q) * VEC + e) * 4, i = q * VEC + e;
      if constexpr (VEC < 4) {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(dw[i]), wr, o, 0, 0);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(db[i]), br, o, 0, 0);
      } else {
        __builtin_amdgcn_raw_buffer_store_b128(
            u32x4_t{__float_as_uint(dw[i]), __float_as_uint(dw[i + 1]), __float_as_uint(dw[i + 2]),
                    __float_as_uint(dw[i + 3])}, wr, o, 0, 0);
        __builtin_amdgcn_raw_buffer_store_b128(
            u32x4_t{__float_as_uint(db[i]), __float_as_uint(db[i + 1]), __float_as_uint(db[i + 2]),
                    __float_as_uint(db[i + 3])}, br, o, 0, 0);
      }
    }
}

constexpr int kSumPitch = 64 + 4;

// Column sums of rows r0 .. r1 of a matrix of fp32 or (uint16_t) bf16, columns
// 64 block ..: thread t has columns 8 (t % 8) .. of every 32nd row; the 32 sums
// are added in order.  The result is that of threads t < 64, for column 64
// block + t.
template <typename X>
__device__ __forceinline__ float column_sum(const X* __restrict__ x, int64_t r0, int64_t r1, int H, int block,
                                            float* s) {
  const int c = threadIdx.x & 7, r = threadIdx.x >> 3;
  const int col = block * 64 + 8 * c;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (col < H) {
#pragma unroll 4
    for (int64_t i = r0 + r; i < r1; i += 32) {
      const u32x4_t u = ld16(x + i * H + col);
      const uint32_t w4[4] = {u.x, u.y, u.z, u.w};
      if constexpr (sizeof(X) == 4) {
        const u32x4_t u2 = ld16(x + i * H + col + 4);
        const uint32_t w8[4] = {u2.x, u2.y, u2.z, u2.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[k] += __uint_as_float(w4[k]);
          v[4 + k] += __uint_as_float(w8[k]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[2 * k] += bf16_bits_to_f32(w4[k] & 0xFFFFu);
          v[2 * k + 1] += bf16_bits_to_f32(w4[k] >> 16);
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) s[r * kSumPitch + 8 * c + k] = v[k];
  __syncthreads();
  if (threadIdx.x >= 64) return 0.f;
  float t = s[threadIdx.x];
#pragma unroll
  for (int i = 1; i < 32; ++i) t += s[i * kSumPitch + threadIdx.x];
  return t;
}

// Partial column sums of two matrices of many rows (the linears' bias gradients:
// dr's, which is there in fp32, and those of dz as the products take it):
// workgroup (x, y, z) has 64 columns of the y-th run of rows of matrix z.  2 x 2049 rows of 2816: 7.6 us (4.6 TB/s).
__global__ __launch_bounds__(256) void k_column_sum(const float* __restrict__ x0, const uint16_t* __restrict__ x1,
                                                    int64_t M, int H, int64_t rows, float* __restrict__ part) {
  __shared__ float s[32 * kSumPitch];
  const int64_t r0 = (int64_t)blockIdx.y * rows;
  const int64_t r1 = min(M, r0 + rows);
  const float t = blockIdx.z == 0 ? column_sum(x0, r0, r1, H, blockIdx.x, s) : column_sum(x1, r0, r1, H, blockIdx.x, s);
  const int o = blockIdx.x * 64 + (int)threadIdx.x;
  if (threadIdx.x < 64 && o < H) part[((int64_t)blockIdx.y * 2 + blockIdx.z) * H + o] = t;
}

// Column sums of partial rows: segment blockIdx.y has nb rows of 2 H floats,
// whose halves, rounded to T, are two gradients (null: not wanted).  A
// workgroup has 32 columns, eight threads a column, each the partials i,
// i + 8, ...; the eight sums are added in order.  A segment with x0 has no
// partials: its gradients are the sums of two matrices of nb rows (32 rows
// of 2816: 4 us less than with a launch of their own).
template <typename T>
__global__ __launch_bounds__(256) void k_column_join(LnJoin a) {
  __shared__ float s[32 * kSumPitch];
  const auto& g = a.seg[blockIdx.y];
  if (std::is_same_v<T, __bf16> && g.x0 != nullptr) {
    const int blocks = (a.H + 63) / 64, z = (int)blockIdx.x >= blocks, block = blockIdx.x - z * blocks;
    if (block >= blocks) return;
    const float t = z ? column_sum(g.x1, 0, g.nb, a.H, block, s) : column_sum(g.x0, 0, g.nb, a.H, block, s);
    const int o = block * 64 + (int)threadIdx.x;
    if (threadIdx.x < 64 && o < a.H) static_cast<T*>(z ? g.out1 : g.out0)[o] = (T)t;
    return;
  }
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), r = threadIdx.x >> 5, cols = 2 * a.H;
  float v = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int i = r; i < g.nb; i += 8) v += g.part[(int64_t)i * cols + c];
  }
  s[threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.x >= 32 || c >= cols) return;
  float t = s[threadIdx.x];
#pragma unroll
  for (int i = 1; i < 8; ++i) t += s[32 * i + threadIdx.x];
  T* o = static_cast<T*>(c < a.H ? g.out0 : g.out1);
  if (o != nullptr) o[c < a.H ? c : c - a.H] = (T)t;
}

namespace {

// the rows that HybridLink's forms take
template <typename T, int VEC>
constexpr bool kLnLink = std::is_same_v<T, __bf16> && VEC > 1;

inline bool ln_vector(const LnArgs& a, int size) {
  const int vec = 16 / size;
  if (a.H % vec != 0) return false;
  const void* p[] = {a.x, a.w, a.b, a.y, a.dy};
  for (const void* q : p)
    if (reinterpret_cast<uintptr_t>(q) & 15u) return false;
  return true;
}

// elements of a row that a wavefront keeps in the backward pass without
// spilling: per lane 48 of 16 bits in pairs, 32 otherwise
template <typename T, int VEC>
constexpr int ln_back_wave_h() {
  return sizeof(T) == 4 || VEC == 1 ? 64 * 32 : 64 * 48;
}

template <typename T, int VEC>
hipError_t ln_forward(const LnArgs& a, hipStream_t s) {
  // few rows: a workgroup each, so that a row's arithmetic is spread out; many:
  // a wavefront each (rows of 2816, workgroup / wavefront: 32 2.8/3.4 us, 512
  // 3.6/3.8, 1024 4.7/4.3, 8192 16.8/13.9)
  const bool wave = a.H <= 64 * 48 && a.M > kLnWaveRows;
  const int per = wave ? 64 : 256;
  const int ept = (a.H + per * VEC - 1) / (per * VEC) * VEC;
  const int64_t groups = wave ? (a.M + 3) / 4 : a.M;
  const dim3 grid((unsigned)std::min<int64_t>(groups, kLnMaxGrid));
#define W4A16_LN1(EPT_, TPR_, FORM_) \
  hipLaunchKernelGGL((k_ln_forward<T, VEC, EPT_, TPR_, FORM_>), grid, dim3(kLnThreads), 0, s, a)
#define W4A16_LN(EPT_, TPR_)                                                           \
  do {                                                                                 \
    if (a.form == kLnPost) {                                                           \
      if constexpr (kLnLink<T, VEC>) W4A16_LN1(EPT_, TPR_, kLnPost);                    \
      else return hipErrorInvalidValue;                                                \
    } else {                                                                           \
      W4A16_LN1(EPT_, TPR_, kLnRows);                                                  \
    }                                                                                  \
  } while (0)
  if (per == 64) {
    if (ept <= 16) W4A16_LN(16, 64);
    else if (ept <= 32) W4A16_LN(32, 64);
    else W4A16_LN(48, 64);
  } else {
    if (ept <= 8) W4A16_LN(8, 256);
    else if (ept <= 16) W4A16_LN(16, 256);
    else W4A16_LN(32, 256);
  }
#undef W4A16_LN
#undef W4A16_LN1
  return hipGetLastError();
}

template <typename T, int VEC>
hipError_t ln_backward(const LnArgs& a, hipStream_t s) {
  if (a.M > 0) {
    // few rows: a workgroup each, one row of partial sums per workgroup; more:
    // wavefronts, whose sums a workgroup joins once (rows of 2816, workgroup /
    // wavefront: 32 3.2/7.6 us, 256 7.1/8.4, 257 9.5/7.9, 4096 22.1/16.1)
    const bool wave = a.H <= ln_back_wave_h<T, VEC>() && a.M > kLnPartials;
    const int per = wave ? 64 : 256;
    const int ept = (a.H + per * VEC - 1) / (per * VEC) * VEC;
    const int nb = ln_partials(a.M);
#define W4A16_LN1(EPT_, TPR_, FORM_)                                                                            \
  hipLaunchKernelGGL((k_ln_backward<T, VEC, EPT_, TPR_, FORM_>), dim3(nb), dim3(ln_back_threads(TPR_)),           \
                     TPR_ == 64 ? 4 * 2 * EPT_ * 64 * 4 : 2 * 4 * 4, s, a)
#define W4A16_LN(EPT_, TPR_)                                                           \
  do {                                                                                 \
    if (a.form != kLnRows) {                                                           \
      if constexpr (!kLnLink<T, VEC>) return hipErrorInvalidValue;                     \
      else if (a.form == kLnPost) W4A16_LN1(EPT_, TPR_, kLnPost);                       \
      else W4A16_LN1(EPT_, TPR_, kLnPre);                                              \
    } else {                                                                           \
      W4A16_LN1(EPT_, TPR_, kLnRows);                                                  \
    }                                                                                  \
  } while (0)
    if (per == 64) {
      if (ept <= 16) W4A16_LN(16, 64);
      else if (ept <= 32) W4A16_LN(32, 64);
      else if constexpr (ln_back_wave_h<T, VEC>() > 64 * 32) W4A16_LN(48, 64);
    } else {
      if (ept <= 16) W4A16_LN(16, 256);
      else W4A16_LN(32, 256);
    }
#undef W4A16_LN
#undef W4A16_LN1
  }
  return hipGetLastError();
}

}  // namespace

int ln_partials(int64_t M) {
  // a workgroup per row, or per eight rows: the wavefront form's at a time, one
  // after another in the workgroup form (rows wider than a wavefront keeps: 256
  // / 257 / 1024 fp32 rows of 2816 6.1/11.2/13.2 us)
  return (int)(M <= kLnPartials ? M : std::min<int64_t>((M + 7) / 8, kLnPartials));
}

hipError_t launch_ln_forward(int dtype, const LnArgs& a, hipStream_t s) {
  if (a.M == 0) return hipSuccess;
  if (a.H <= 0 || a.H > kLnMaxH) return hipErrorInvalidValue;
  const bool v = ln_vector(a, dtype == 2 ? 4 : 2);
  switch (dtype) {
    case 0: return v ? ln_forward<__bf16, 8>(a, s) : ln_forward<__bf16, 1>(a, s);
    case 1: return v ? ln_forward<_Float16, 8>(a, s) : ln_forward<_Float16, 1>(a, s);
    case 2: return v ? ln_forward<float, 4>(a, s) : ln_forward<float, 1>(a, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_ln_backward(int dtype, const LnArgs& a, hipStream_t s) {
  if (a.H <= 0 || a.H > kLnMaxH || a.M < 0) return hipErrorInvalidValue;
  const bool v = ln_vector(a, dtype == 2 ? 4 : 2);
  switch (dtype) {
    case 0: return v ? ln_backward<__bf16, 8>(a, s) : ln_backward<__bf16, 1>(a, s);
    case 1: return v ? ln_backward<_Float16, 8>(a, s) : ln_backward<_Float16, 1>(a, s);
    case 2: return v ? ln_backward<float, 4>(a, s) : ln_backward<float, 1>(a, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_column_join(int dtype, const LnJoin& a, hipStream_t s) {
  if (a.n == 0) return hipSuccess;
  const dim3 grid((2 * a.H + 31) / 32, a.n);
  switch (dtype) {
    case 0: hipLaunchKernelGGL(k_column_join<__bf16>, grid, dim3(256), 0, s, a); break;
    case 1: hipLaunchKernelGGL(k_column_join<_Float16>, grid, dim3(256), 0, s, a); break;
    case 2: hipLaunchKernelGGL(k_column_join<float>, grid, dim3(256), 0, s, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

int column_sum_partials(int64_t M) {
  return M <= kColSumRows ? 0 : (int)std::min<int64_t>((M + kColSumRows - 1) / kColSumRows, kColSumPartials);
}

hipError_t launch_column_sums(const float* x0, const uint16_t* x1, int64_t M, int H, float* part, hipStream_t s) {
  const int n = column_sum_partials(M);
  if (H <= 0 || H % 8 != 0 || n <= 0) return hipErrorInvalidValue;
  hipLaunchKernelGGL(k_column_sum, dim3((H + 63) / 64, n, 2), dim3(256), 0, s, x0, x1, M, H, (M + n - 1) / n, part);
  return hipGetLastError();
}

}  // namespace w4a16
