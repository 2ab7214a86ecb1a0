// C ABI of the training forms: layer norm, the gated MLP and HybridLink with
// their backward passes (include/w4a16moe.h states each contract).
#include "w4a16moe.h"

#include <algorithm>

#include "launch.hpp"
#include "rules.hpp"

using namespace w4a16;

namespace {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline size_t round256(size_t b) { return (b + 255) & ~size_t(255); }
inline int launch_status(hipError_t e) { return e == hipSuccess ? W4A16_OK : W4A16_ERR_LAUNCH; }

constexpr int64_t kMaxRows = (int64_t(1) << 24) - 1;
constexpr int64_t kMaxWidth = 32768;

// Bump allocator over a caller-provided buffer.
struct Carve {
  char* base;
  size_t used = 0;
  explicit Carve(void* p) : base(static_cast<char*>(p)) {}
  template <typename T>
  T* take(size_t count) {
    T* p = reinterpret_cast<T*>(base ? base + used : nullptr);
    used += round256(count * sizeof(T));
    return p;
  }
};

// floats of partial sums that a product of `plane` elements may be split into
inline size_t part_floats(int64_t plane) {
  const int n = dense_part_planes(plane);
  return n > 1 ? (size_t)n * plane : 0;
}

inline bool bad_matrix(int64_t n) { return n <= 0 || n % 32 != 0 || n > kMaxWidth; }

inline DgProblem problem(const uint16_t* A, int64_t lda, const uint16_t* B, int64_t ldb, int64_t M, int64_t N,
                         const DgEpilogue& e) {
  DgProblem p{};
  p.A = A;
  p.B = B;
  p.M = (int)M;
  p.N = (int)N;
  p.lda = (int)lda;
  p.ldb = (int)ldb;
  p.e = e;
  return p;
}

inline DgEpilogue to(uint16_t* out) { return DgEpilogue{out, nullptr, nullptr, nullptr, nullptr, nullptr}; }

inline hipError_t product(int layout, int epi, const DgProblem& p, int64_t K, float* part, hipStream_t s) {
  DgArgs a{};
  a.prob[0] = p;
  a.nprob = 1;
  a.K = (int)K;
  a.part = part_floats((int64_t)p.M * p.N * (epi == kDgGateUp ? 2 : 1)) > 0 ? part : nullptr;
  return launch_gemm_dense(layout, epi, a, s);
}

struct MlpSaved {
  float *gate, *up;
  uint16_t* inter;
  size_t bytes;
};
MlpSaved mlp_saved(void* p, int64_t M, int64_t I) {
  Carve c(p);
  MlpSaved s;
  s.gate = c.take<float>(M * I);
  s.up = c.take<float>(M * I);
  s.inter = c.take<uint16_t>(M * I);
  s.bytes = c.used;
  return s;
}

struct MlpWs {
  uint16_t* inter;
  float* part;
  size_t bytes;
};
MlpWs mlp_ws(void* p, int64_t M, int64_t H, int64_t I) {
  Carve c(p);
  MlpWs w;
  w.inter = c.take<uint16_t>(M * I);
  w.part = c.take<float>(std::max(part_floats(2 * M * I), part_floats(M * H)));
  w.bytes = c.used;
  return w;
}

struct MlpBackWs {
  uint16_t *da, *db;
  float* part;
  size_t bytes;
};
MlpBackWs mlp_back_ws(void* p, int64_t M, int64_t H, int64_t I) {
  Carve c(p);
  MlpBackWs w;
  w.da = c.take<uint16_t>(M * I);
  w.db = c.take<uint16_t>(M * I);
  w.part = c.take<float>(std::max({part_floats(M * I), part_floats(M * H), part_floats(H * I), part_floats(2 * H * I),
                                   part_floats(3 * H * I)}));
  w.bytes = c.used;
  return w;
}

// HybridLink's tensors between the kernels: a, g, dr and dz are operands of the
// bf16 matrix instructions and rounded once each, from fp32.  z, r and da, which
// an activation or a norm reads, and dr where it is the residual's gradient or
// summed, stay in fp32 (2049 rows of 2816: 17 us of a step of 280; rounded to
// bf16, r alone would lose what proj2 adds to a row far from zero).  Against 64
// bits (Frobenius norm, the same rows) out is 0.0021 off and the gradients
// 0.0017 .. 0.0036, a single rounding 0.0017.
struct LinkSaved {
  uint16_t *a, *g;
  float *z, *r;
  float *mean1, *rstd1, *mean2, *rstd2;
  size_t bytes;
};
LinkSaved link_saved(void* p, int64_t B, int64_t H) {
  Carve c(p);
  LinkSaved s;
  s.a = c.take<uint16_t>(B * H);
  s.g = c.take<uint16_t>(B * H);
  s.z = c.take<float>(B * H);
  s.r = c.take<float>(B * H);
  s.mean1 = c.take<float>(B);
  s.rstd1 = c.take<float>(B);
  s.mean2 = c.take<float>(B);
  s.rstd2 = c.take<float>(B);
  s.bytes = c.used;
  return s;
}

struct LinkBackWs {
  uint16_t *dr, *dz;
  float *dr32, *da;
  float *part, *ln2, *ln1, *cols;
  size_t bytes;
};
LinkBackWs link_back_ws(void* p, int64_t B, int64_t H) {
  Carve c(p);
  LinkBackWs w;
  w.dr = c.take<uint16_t>(B * H);
  w.dz = c.take<uint16_t>(B * H);
  w.dr32 = c.take<float>(B * H);
  w.da = c.take<float>(B * H);
  w.part = c.take<float>(std::max(part_floats(B * H), part_floats(2 * H * H)));
  // partial rows of the column sums, added in one launch at the end
  w.ln2 = c.take<float>((size_t)ln_partials(B) * 2 * H);
  w.ln1 = c.take<float>((size_t)ln_partials(B) * 2 * H);
  w.cols = c.take<float>((size_t)column_sum_partials(B) * 2 * H);
  w.bytes = c.used;
  return w;
}

inline LnArgs ln_args(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t M,
                      int64_t H, float eps) {
  LnArgs a{};
  a.x = x;
  a.w = w;
  a.b = b;
  a.y = y;
  a.mean = mean;
  a.rstd = rstd;
  a.M = M;
  a.H = (int)H;
  a.eps = eps;
  return a;
}

}  // namespace

extern "C" {

int w4a16_layer_norm(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, int dtype,
                     int64_t M, int64_t H, float eps, void* stream) {
  if (M < 0 || M > kMaxRows || H <= 0 || H > kLnMaxH || dtype < W4A16_BF16 || dtype > W4A16_F32)
    return W4A16_ERR_SHAPE;
  if (M == 0) return W4A16_OK;
  if (!x || !weight || !y || (mean == nullptr) != (rstd == nullptr)) return W4A16_ERR_NULL;
  return launch_status(launch_ln_forward(dtype, ln_args(x, weight, bias, y, mean, rstd, M, H, eps),
                                         static_cast<hipStream_t>(stream)));
}

size_t w4a16_layer_norm_backward_workspace_bytes(int64_t M, int64_t H) {
  if (M <= 0 || H <= 0) return 0;
  return round256((size_t)ln_partials(M) * 2 * H * sizeof(float));
}

int w4a16_layer_norm_backward(const void* dy, const void* x, const void* weight, const float* mean, const float* rstd,
                              void* dx, void* dweight, void* dbias, int dtype, int64_t M, int64_t H, void* workspace,
                              size_t workspace_bytes, void* stream) {
  if (M < 0 || M > kMaxRows || H <= 0 || H > kLnMaxH || dtype < W4A16_BF16 || dtype > W4A16_F32)
    return W4A16_ERR_SHAPE;
  if (!dweight || (M > 0 && (!dy || !x || !weight || !mean || !rstd || !dx))) return W4A16_ERR_NULL;
  if (M > 0 && (workspace == nullptr || workspace_bytes < w4a16_layer_norm_backward_workspace_bytes(M, H)))
    return W4A16_ERR_WORKSPACE;
  if (!aligned16(workspace)) return W4A16_ERR_ALIGN;
  LnArgs a = ln_args(x, weight, nullptr, dx, const_cast<float*>(mean), const_cast<float*>(rstd), M, H, 0.f);
  a.dy = dy;
  a.part = static_cast<float*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  LnJoin j{};
  j.seg[0] = {a.part, ln_partials(M), dweight, dbias};
  j.n = 1;
  j.H = (int)H;
  hipError_t e = launch_ln_backward(dtype, a, s);
  if (e == hipSuccess) e = launch_column_join(dtype, j, s);
  return launch_status(e);
}

size_t w4a16_gated_mlp_workspace_bytes(int64_t M, int64_t H, int64_t I) {
  if (M <= 0 || H <= 0 || I <= 0) return 0;
  return mlp_ws(nullptr, M, H, I).bytes;
}

size_t w4a16_gated_mlp_saved_bytes(int64_t M, int64_t I) {
  if (M <= 0 || I <= 0) return 0;
  return mlp_saved(nullptr, M, I).bytes;
}

int w4a16_gated_mlp(const uint16_t* x, const uint16_t* gate_w, const uint16_t* up_w, const uint16_t* down_w,
                    uint16_t* y, void* saved, size_t saved_bytes, int64_t M, int64_t H, int64_t I, void* workspace,
                    size_t workspace_bytes, void* stream) {
  if (M < 0 || M > kMaxRows || bad_matrix(H) || bad_matrix(I)) return W4A16_ERR_SHAPE;
  if (M == 0) return W4A16_OK;
  if (!x || !gate_w || !up_w || !down_w || !y) return W4A16_ERR_NULL;
  if (!aligned16(x) || !aligned16(gate_w) || !aligned16(up_w) || !aligned16(down_w) || !aligned16(y) ||
      !aligned16(saved) || !aligned16(workspace))
    return W4A16_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < w4a16_gated_mlp_workspace_bytes(M, H, I) ||
      (saved != nullptr && saved_bytes < w4a16_gated_mlp_saved_bytes(M, I)))
    return W4A16_ERR_WORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const MlpWs ws = mlp_ws(workspace, M, H, I);
  DgEpilogue e = to(ws.inter);
  if (saved != nullptr) {
    const MlpSaved sv = mlp_saved(saved, M, I);
    e = DgEpilogue{sv.inter, nullptr, sv.gate, sv.up, nullptr, nullptr};
  }
  DgProblem p = problem(x, H, gate_w, H, M, I, e);
  p.B2 = up_w;
  hipError_t st = product(kDgNT, kDgGateUp, p, H, ws.part, s);
  if (st == hipSuccess) st = product(kDgNT, kDgPlain, problem(e.out, I, down_w, I, M, H, to(y)), I, ws.part, s);
  return launch_status(st);
}

size_t w4a16_gated_mlp_backward_workspace_bytes(int64_t M, int64_t H, int64_t I) {
  if (M <= 0 || H <= 0 || I <= 0) return 0;
  return mlp_back_ws(nullptr, M, H, I).bytes;
}

int w4a16_gated_mlp_backward(const uint16_t* dy, const uint16_t* x, const uint16_t* gate_w, const uint16_t* up_w,
                             const uint16_t* down_w, const void* saved, size_t saved_bytes, uint16_t* dx,
                             uint16_t* dgate_w, uint16_t* dup_w, uint16_t* ddown_w, int64_t M, int64_t H, int64_t I,
                             void* workspace, size_t workspace_bytes, void* stream) {
  if (M < 0 || M > kMaxRows || bad_matrix(H) || bad_matrix(I)) return W4A16_ERR_SHAPE;
  if (M > 0 && (!dy || !x || !gate_w || !up_w || !down_w || !saved)) return W4A16_ERR_NULL;
  const void* a16[] = {dy, x, gate_w, up_w, down_w, saved, dx, dgate_w, dup_w, ddown_w, workspace};
  for (const void* p : a16)
    if (!aligned16(p)) return W4A16_ERR_ALIGN;
  if (M > 0 && (workspace == nullptr || workspace_bytes < w4a16_gated_mlp_backward_workspace_bytes(M, H, I) ||
                saved_bytes < w4a16_gated_mlp_saved_bytes(M, I)))
    return W4A16_ERR_WORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const MlpSaved sv = mlp_saved(const_cast<void*>(saved), M, I);
  const MlpBackWs ws = mlp_back_ws(M > 0 ? workspace : nullptr, M, H, I);
  hipError_t st = hipSuccess;
  // dh = dy Wd; da, db
  if (M > 0 && (dx || dgate_w || dup_w))
    st = product(kDgNN, kDgGateUpBack,
                 problem(dy, H, down_w, I, M, I, DgEpilogue{ws.da, ws.db, sv.gate, sv.up, nullptr, nullptr}), H,
                 ws.part, s);
  if (st == hipSuccess && M > 0 && dx) {
    // dx = da Wg + db Wu
    DgProblem p = problem(ws.da, I, gate_w, H, M, H, to(dx));
    p.A2 = ws.db;
    p.B2 = up_w;
    st = product(kDgNN, kDgPlain, p, I, ws.part, s);
  }
  DgArgs a{};
  if (ddown_w) a.prob[a.nprob++] = problem(dy, H, sv.inter, I, H, I, to(ddown_w));
  if (dgate_w) a.prob[a.nprob++] = problem(ws.da, I, x, H, I, H, to(dgate_w));
  if (dup_w) a.prob[a.nprob++] = problem(ws.db, I, x, H, I, H, to(dup_w));
  if (st == hipSuccess && a.nprob > 0) {
    a.K = (int)M;
    a.part = M > 0 && part_floats(a.nprob * H * I) > 0 ? ws.part : nullptr;
    st = launch_gemm_dense(kDgTN, kDgPlain, a, s);
  }
  return launch_status(st);
}

size_t w4a16_hybridlink_saved_bytes(int64_t B, int64_t H) {
  if (B <= 0 || H <= 0) return 0;
  return link_saved(nullptr, B, H).bytes;
}

size_t w4a16_hybridlink_train_workspace_bytes(int64_t B, int64_t H) {
  if (B <= 0 || H <= 0) return 0;
  return round256(part_floats(B * H) * sizeof(float));
}

int w4a16_hybridlink_train(const uint16_t* h, const uint16_t* ln1_w, const uint16_t* ln1_b, const uint16_t* p1_w,
                           const uint16_t* p1_b, const uint16_t* p2_w, const uint16_t* p2_b, const uint16_t* ln2_w,
                           const uint16_t* ln2_b, uint16_t* out, void* saved, size_t saved_bytes, int64_t B, int64_t H,
                           float eps, void* workspace, size_t workspace_bytes, void* stream) {
  if (B < 0 || B > kMaxRows || H <= 0 || H % 32 != 0 || H > kLnMaxH) return W4A16_ERR_SHAPE;
  if (B == 0) return W4A16_OK;
  if (!h || !ln1_w || !ln1_b || !p1_w || !p1_b || !p2_w || !p2_b || !ln2_w || !ln2_b || !out || !saved)
    return W4A16_ERR_NULL;
  const void* a16[] = {h, ln1_w, ln1_b, p1_w, p1_b, p2_w, p2_b, ln2_w, ln2_b, out, saved, workspace};
  for (const void* p : a16)
    if (!aligned16(p)) return W4A16_ERR_ALIGN;
  const size_t need = w4a16_hybridlink_train_workspace_bytes(B, H);
  if (saved_bytes < w4a16_hybridlink_saved_bytes(B, H) || (need > 0 && (workspace == nullptr || workspace_bytes < need)))
    return W4A16_ERR_WORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const LinkSaved sv = link_saved(saved, B, H);
  float* part = need > 0 ? static_cast<float*>(workspace) : nullptr;
  hipError_t e = launch_ln_forward(W4A16_BF16, ln_args(h, ln1_w, ln1_b, sv.a, sv.mean1, sv.rstd1, B, H, eps), s);
  if (e == hipSuccess)
    e = product(kDgNT, kDgBiasGelu,
                problem(sv.a, H, p1_w, H, B, H, DgEpilogue{sv.g, nullptr, sv.z, nullptr, nullptr, p1_b}), H, part, s);
  if (e == hipSuccess)
    e = product(kDgNT, kDgBiasResidual,
                problem(sv.g, H, p2_w, H, B, H, DgEpilogue{nullptr, nullptr, sv.r, nullptr, h, p2_b}), H, part, s);
  LnArgs n2 = ln_args(sv.r, ln2_w, ln2_b, out, sv.mean2, sv.rstd2, B, H, eps);
  n2.form = kLnPost;
  if (e == hipSuccess) e = launch_ln_forward(W4A16_BF16, n2, s);
  return launch_status(e);
}

size_t w4a16_hybridlink_backward_workspace_bytes(int64_t B, int64_t H) {
  if (B <= 0 || H <= 0) return 0;
  return link_back_ws(nullptr, B, H).bytes;
}

int w4a16_hybridlink_backward(const uint16_t* dout, const uint16_t* h, const uint16_t* ln1_w, const uint16_t* p1_w,
                              const uint16_t* p2_w, const uint16_t* ln2_w, const void* saved, size_t saved_bytes,
                              uint16_t* dh, uint16_t* dln1_w, uint16_t* dln1_b, uint16_t* dp1_w, uint16_t* dp1_b,
                              uint16_t* dp2_w, uint16_t* dp2_b, uint16_t* dln2_w, uint16_t* dln2_b, int64_t B,
                              int64_t H, void* workspace, size_t workspace_bytes, void* stream) {
  if (B < 0 || B > kMaxRows || H <= 0 || H % 32 != 0 || H > kLnMaxH) return W4A16_ERR_SHAPE;
  if (!dln1_w || !dln1_b || !dp1_w || !dp1_b || !dp2_w || !dp2_b || !dln2_w || !dln2_b) return W4A16_ERR_NULL;
  if (B > 0 && (!dout || !h || !ln1_w || !p1_w || !p2_w || !ln2_w || !saved || !dh)) return W4A16_ERR_NULL;
  const void* a16[] = {dout, h, ln1_w, p1_w, p2_w, ln2_w, saved, dh, dln1_w, dln1_b, dp1_w, dp1_b, dp2_w, dp2_b,
                       dln2_w, dln2_b, workspace};
  for (const void* p : a16)
    if (!aligned16(p)) return W4A16_ERR_ALIGN;
  if (B > 0 && (workspace == nullptr || workspace_bytes < w4a16_hybridlink_backward_workspace_bytes(B, H) ||
                saved_bytes < w4a16_hybridlink_saved_bytes(B, H)))
    return W4A16_ERR_WORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const LinkSaved sv = link_saved(const_cast<void*>(saved), B, H);
  const LinkBackWs ws = link_back_ws(B > 0 ? workspace : nullptr, B, H);
  // post_ln: dr, the gradient of r = h + proj2(g)
  LnArgs n2 = ln_args(sv.r, ln2_w, nullptr, ws.dr, sv.mean2, sv.rstd2, B, H, 0.f);
  n2.form = kLnPost;
  n2.y32 = ws.dr32;
  n2.dy = dout;
  n2.part = ws.ln2;
  hipError_t e = launch_ln_backward(W4A16_BF16, n2, s);
  // dz = (dr W2) gelu'(z), da = dz W1
  if (e == hipSuccess && B > 0)
    e = product(kDgNN, kDgGeluBack,
                problem(ws.dr, H, p2_w, H, B, H, DgEpilogue{ws.dz, nullptr, sv.z, nullptr, nullptr, nullptr}), H,
                ws.part, s);
  if (e == hipSuccess && B > 0)
    e = product(kDgNN, kDgSums,
                problem(ws.dz, H, p1_w, H, B, H, DgEpilogue{nullptr, nullptr, ws.da, nullptr, nullptr, nullptr}), H,
                ws.part, s);
  if (e == hipSuccess) {
    DgArgs a{};
    a.prob[0] = problem(ws.dr, H, sv.g, H, H, H, to(dp2_w));
    a.prob[1] = problem(ws.dz, H, sv.a, H, H, H, to(dp1_w));
    a.nprob = 2;
    a.K = (int)B;
    a.part = B > 0 && part_floats(2 * H * H) > 0 ? ws.part : nullptr;
    e = launch_gemm_dense(kDgTN, kDgPlain, a, s);
  }
  const int sums = column_sum_partials(B);
  if (e == hipSuccess && sums > 0) e = launch_column_sums(ws.dr32, ws.dz, B, (int)H, ws.cols, s);
  // pre_ln, and the residual's dr
  LnArgs n1 = ln_args(h, ln1_w, nullptr, dh, sv.mean1, sv.rstd1, B, H, 0.f);
  n1.form = kLnPre;
  n1.dy = ws.da;
  n1.add = ws.dr32;
  n1.part = ws.ln1;
  if (e == hipSuccess) e = launch_ln_backward(W4A16_BF16, n1, s);
  LnJoin j{};
  j.seg[0] = {ws.ln1, ln_partials(B), dln1_w, dln1_b, nullptr, nullptr};
  j.seg[1] = {ws.ln2, ln_partials(B), dln2_w, dln2_b, nullptr, nullptr};
  if (sums > 0 || B == 0)
    j.seg[2] = {ws.cols, sums, dp2_b, dp1_b, nullptr, nullptr};
  else
    j.seg[2] = {nullptr, (int)B, dp2_b, dp1_b, ws.dr32, ws.dz};
  j.n = 3;
  j.H = (int)H;
  if (e == hipSuccess) e = launch_column_join(W4A16_BF16, j, s);
  return launch_status(e);
}

}  // extern "C"
