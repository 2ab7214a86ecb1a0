// C ABI of the attention half of a decoder layer: the heads' norms with the
// position rotation, the paged key-value cache, attention over packed prompts
// with its gradients and over the cache (include/w4a16moe.h states each contract).
#include "w4a16moe.h"

#include <algorithm>
#include <cmath>

#include "launch.hpp"

using namespace w4a16;

namespace {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline int launch_status(hipError_t e) { return e == hipSuccess ? W4A16_OK : W4A16_ERR_LAUNCH; }

constexpr int64_t kMaxTokens = (int64_t(1) << 24) - 1;
constexpr int64_t kMaxHeads = 1024;
constexpr int64_t kMaxSequences = 1 << 14;  // every workgroup goes through their lengths
constexpr int64_t kMaxBlocks = (int64_t(1) << 24) - 1;  // 256 threads each: a launch has 2^32 at most
// bytes between two tokens, between two heads: a tile of 32 rows is addressed in 32 bits
constexpr int64_t kMaxStride = int64_t(1) << 26;

// [tokens][heads][D] with any strides that keep the rows 16-byte aligned
struct Heads {
  const void* p;
  int64_t token, head;
};
inline int64_t size_of(int dtype) { return dtype == W4A16_F32 ? 4 : 2; }
inline bool bad_stride(const Heads& h, int64_t size) {
  return h.token < 0 || h.head < 0 || h.token * size > kMaxStride || h.head * size > kMaxStride;
}
inline bool odd(const Heads& h, int64_t size) {
  return !aligned16(h.p) || (h.token * size) % 16 != 0 || (h.head * size) % 16 != 0;
}
inline bool bad_heads(int64_t Hq, int64_t Hk) { return Hq <= 0 || Hk <= 0 || Hq > kMaxHeads || Hk > kMaxHeads; }
inline bool bad_group(int64_t Hq, int64_t Hk) { return bad_heads(Hq, Hk) || Hq % Hk != 0; }
inline bool bad_attn_dim(int64_t D) { return D != 64 && D != 128 && D != 256 && D != 512; }
inline bool bad_scale(float scale) { return !(scale > 0.f) || !std::isfinite(scale); }

// what the three forms of the heads' norm check alike
int head_norm_args(HeadNormArgs& a, const Heads& q, const Heads& k, const Heads& v, const float* cos, const float* sin,
                   const int32_t* pos, const void* qw, const void* kw, int dtype, int64_t T, int64_t Hq, int64_t Hk,
                   int64_t D, int64_t P, int64_t R, float eps) {
  if (T < 0 || T > kMaxTokens || bad_heads(Hq, Hk) || D <= 0 || D % 8 != 0 || D > kHeadNormMaxD || R < 0 ||
      R % 8 != 0 || R > D || (R > 0 && P <= 0) || P < 0 || P > INT32_MAX || !(eps >= 0.f))
    return W4A16_ERR_SHAPE;
  const int64_t size = size_of(dtype);
  if (bad_stride(q, size) || bad_stride(k, size) || (v.p && bad_stride(v, size))) return W4A16_ERR_SHAPE;
  // a wavefront takes one row at least
  if ((T * (Hq + 2 * Hk) + 3) / 4 > kMaxBlocks) return W4A16_ERR_SHAPE;
  if ((qw == nullptr) != (kw == nullptr)) return W4A16_ERR_NULL;
  if (T > 0 && (!q.p || !k.p || !pos || (R > 0 && (!cos || !sin)))) return W4A16_ERR_NULL;
  if (odd(q, size) || odd(k, size) || (v.p && odd(v, size)) || !aligned16(cos) || !aligned16(sin) || !aligned16(qw) ||
      !aligned16(kw))
    return W4A16_ERR_ALIGN;
  a = HeadNormArgs{};
  a.q = q.p;
  a.k = k.p;
  a.v = v.p;
  a.q_tok = q.token * size;
  a.q_head = q.head * size;
  a.k_tok = k.token * size;
  a.k_head = k.head * size;
  a.v_tok = v.token * size;
  a.v_head = v.head * size;
  a.cos = cos;
  a.sin = sin;
  a.pos = pos;
  a.qw = qw;
  a.kw = kw;
  a.T = (int)T;
  a.Hq = (int)Hq;
  a.Hk = (int)Hk;
  a.D = (int)D;
  a.P = R > 0 ? (int)P : INT32_MAX;
  a.R = (int)R;
  a.v_norm = true;
  a.eps = eps;
  return W4A16_OK;
}

int attn_args(AttnArgs& a, const Heads& q, const Heads& k, const Heads& v, const int32_t* cu_q, const int32_t* cu_k,
              int dtype, int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D, float scale, int causal,
              int64_t window) {
  if ((dtype != W4A16_BF16 && dtype != W4A16_F16) || B < 0 || B > kMaxSequences || Tq < 0 || Tq > kMaxTokens ||
      Tk < 0 || Tk > kMaxTokens || bad_group(Hq, Hk) || bad_attn_dim(D) || bad_scale(scale) || window < 0 ||
      (window > 0 && !causal) || bad_stride(q, 2) || bad_stride(k, 2) || bad_stride(v, 2))
    return W4A16_ERR_SHAPE;
  // workgroups of 64 rows at least and 512 threads
  if ((std::max(Tq, Tk) / 64 + B + 9) * Hq > kMaxBlocks / 2) return W4A16_ERR_SHAPE;
  if ((Tq > 0 && !q.p) || (Tk > 0 && (!k.p || !v.p)) || !cu_q || !cu_k) return W4A16_ERR_NULL;
  if (odd(q, 2) || odd(k, 2) || odd(v, 2)) return W4A16_ERR_ALIGN;
  a = AttnArgs{};
  a.q = q.p;
  a.k = k.p;
  a.v = v.p;
  a.q_stride = 2 * q.token;
  a.q_head = 2 * q.head;
  a.k_stride = 2 * k.token;
  a.k_head = 2 * k.head;
  a.v_stride = 2 * v.token;
  a.v_head = 2 * v.head;
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.B = (int)B;
  a.Tq = (int)Tq;
  a.Tk = (int)Tk;
  a.Hq = (int)Hq;
  a.Hk = (int)Hk;
  a.group = (int)(Hq / Hk);
  a.D = (int)D;
  a.scale = scale;
  a.scale2 = scale * 1.4426950408889634f;
  a.window = (int)std::min<int64_t>(window, kMaxTokens + 1);
  a.causal = causal != 0;
  return W4A16_OK;
}

// bytes of the backward pass' workspace: delta, then the parts of one split kernel
inline size_t delta_floats(int64_t Tq, int64_t Hq) { return ((size_t)Tq * Hq + 3) & ~size_t(3); }

inline int log2_of(int64_t n) {
  int i = 0;
  while ((int64_t(1) << i) < n) ++i;
  return i;
}
inline bool bad_page(int64_t n) { return n < 16 || n > 1024 || (n & (n - 1)) != 0; }

}  // namespace

extern "C" {

int w4a16_head_norm_rope(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token,
                         int64_t k_head, const void* v, int64_t v_token, int64_t v_head, const float* cos,
                         const float* sin, const int32_t* positions, const void* q_weight, const void* k_weight,
                         void* q_out, void* k_out, void* v_out, int dtype, int64_t T, int64_t Hq, int64_t Hk,
                         int64_t D, int64_t P, int64_t R, float eps, void* stream) {
  if (dtype < W4A16_BF16 || dtype > W4A16_F32) return W4A16_ERR_SHAPE;
  HeadNormArgs a;
  const int st = head_norm_args(a, {q, q_token, q_head}, {k, k_token, k_head}, {v, v_token, v_head}, cos, sin,
                                positions, q_weight, k_weight, dtype, T, Hq, Hk, D, P, R, eps);
  if (st != W4A16_OK) return st;
  if (T == 0) return W4A16_OK;
  if (!q_out || !k_out || (v && !v_out)) return W4A16_ERR_NULL;
  if (!aligned16(q_out) || !aligned16(k_out) || !aligned16(v_out)) return W4A16_ERR_ALIGN;
  a.yq = q_out;
  a.yk = k_out;
  a.yv = v_out;
  return launch_status(launch_head_norm(dtype, false, a, static_cast<hipStream_t>(stream)));
}

size_t w4a16_head_norm_rope_backward_workspace_bytes(int64_t T, int64_t Hq, int64_t Hk, int64_t D) {
  if (T <= 0 || Hq <= 0 || Hk <= 0 || D <= 0) return 0;
  return (size_t)head_norm_partials(T, Hq + 2 * Hk, D) * 2 * D * sizeof(float);
}

int w4a16_head_norm_rope_backward(const void* dq, const void* dk, const void* dv, const void* q, int64_t q_token,
                                  int64_t q_head, const void* k, int64_t k_token, int64_t k_head, const void* v,
                                  int64_t v_token, int64_t v_head, const float* cos, const float* sin,
                                  const int32_t* positions, const void* q_weight, const void* k_weight, void* dq_in,
                                  void* dk_in, void* dv_in, void* dq_weight, void* dk_weight, int dtype, int64_t T,
                                  int64_t Hq, int64_t Hk, int64_t D, int64_t P, int64_t R, float eps, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (dtype < W4A16_BF16 || dtype > W4A16_F32) return W4A16_ERR_SHAPE;
  HeadNormArgs a;
  const int st = head_norm_args(a, {q, q_token, q_head}, {k, k_token, k_head}, {v, v_token, v_head}, cos, sin,
                                positions, q_weight, k_weight, dtype, T, Hq, Hk, D, P, R, eps);
  if (st != W4A16_OK) return st;
  const bool weights = dq_weight != nullptr || dk_weight != nullptr;
  if (weights && (!dq_weight || !dk_weight || (T > 0 && !q_weight))) return W4A16_ERR_NULL;
  if (T > 0 && (!dq || !dk || (v && !dv) || !dq_in || !dk_in || (v && !dv_in))) return W4A16_ERR_NULL;
  const void* p[] = {dq, dk, dv, dq_in, dk_in, dv_in, workspace};
  for (const void* x : p)
    if (!aligned16(x)) return W4A16_ERR_ALIGN;
  const size_t need = weights ? w4a16_head_norm_rope_backward_workspace_bytes(T, Hq, Hk, D) : 0;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return W4A16_ERR_WORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.yq = dq_in;
  a.yk = dk_in;
  a.yv = dv_in;
  a.part = weights ? static_cast<float*>(workspace) : nullptr;
  hipError_t e = hipSuccess;
  if (T > 0) e = launch_head_norm_backward(dtype, a, s);
  if (e == hipSuccess && weights) {
    LnJoin j{};
    j.seg[0] = {a.part, T > 0 ? head_norm_partials(T, Hq + (v ? 2 : 1) * Hk, D) : 0, dq_weight, dk_weight};
    j.n = 1;
    j.H = (int)D;
    e = launch_column_join(dtype, j, s);
  }
  return launch_status(e);
}

int w4a16_append_kv(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                    const void* v, int64_t v_token, int64_t v_head, const float* cos, const float* sin,
                    const int32_t* positions, const int32_t* slots, const void* q_weight, const void* k_weight,
                    void* q_out, void* k_out, void* v_out, void* k_cache, int64_t k_page_stride, void* v_cache,
                    int64_t v_page_stride, int dtype, int v_norm, int64_t T, int64_t Hq, int64_t Hk, int64_t D,
                    int64_t P, int64_t R, int64_t pages, int64_t page_size, float eps, void* stream) {
  if (dtype != W4A16_BF16 && dtype != W4A16_F16) return W4A16_ERR_SHAPE;
  HeadNormArgs a;
  const int st = head_norm_args(a, {q, q_token, q_head}, {k, k_token, k_head}, {v, v_token, v_head}, cos, sin,
                                positions, q_weight, k_weight, dtype, T, Hq, Hk, D, P, R, eps);
  if (st != W4A16_OK) return st;
  if (bad_page(page_size) || pages <= 0 || pages * page_size > INT32_MAX || k_page_stride < Hk * page_size * D ||
      v_page_stride < Hk * page_size * D)
    return W4A16_ERR_SHAPE;
  if (T == 0) return W4A16_OK;
  if (!v || !slots || !q_out || !k_cache || !v_cache || (k_out == nullptr) != (v_out == nullptr)) return W4A16_ERR_NULL;
  if (!aligned16(q_out) || !aligned16(k_out) || !aligned16(v_out) || !aligned16(k_cache) || !aligned16(v_cache) ||
      k_page_stride % 8 != 0 || v_page_stride % 8 != 0)
    return W4A16_ERR_ALIGN;
  a.yq = q_out;
  a.yk = k_out;
  a.yv = v_out;
  a.kc = k_cache;
  a.vc = v_cache;
  a.k_page = 2 * k_page_stride;
  a.v_page = 2 * v_page_stride;
  a.slots = slots;
  a.page = (int)page_size;
  a.slots_n = (int)(pages * page_size);
  a.v_norm = v_norm != 0;
  return launch_status(launch_head_norm(dtype, true, a, static_cast<hipStream_t>(stream)));
}

size_t w4a16_attention_workspace_bytes(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D,
                                       int64_t window) {
  if (B <= 0 || Tq <= 0 || Tk <= 0 || bad_group(Hq, Hk) || bad_attn_dim(D) || window < 0) return 0;
  return attn_split(kAttnForward, B, Tq, Tk, Hq, Hk, D, window).floats * sizeof(float);
}

int w4a16_attention(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                    const void* v, int64_t v_token, int64_t v_head, const int32_t* cu_q, const int32_t* cu_k, void* out,
                    float* lse, int dtype, int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D,
                    float scale, int causal, int64_t window, void* workspace, size_t workspace_bytes, void* stream) {
  AttnArgs a;
  const int st = attn_args(a, {q, q_token, q_head}, {k, k_token, k_head}, {v, v_token, v_head}, cu_q, cu_k, dtype, B,
                           Tq, Tk, Hq, Hk, D, scale, causal, window);
  if (st != W4A16_OK) return st;
  if (Tq == 0) return W4A16_OK;
  if (!out) return W4A16_ERR_NULL;
  if (!aligned16(out) || !aligned16(workspace)) return W4A16_ERR_ALIGN;
  const AttnSplit p = attn_split(kAttnForward, B, Tq, Tk, Hq, Hk, D, window);
  if (p.floats > 0 && (workspace == nullptr || workspace_bytes < p.floats * sizeof(float))) return W4A16_ERR_WORKSPACE;
  a.out = out;
  a.lse = lse;
  a.low = p.low;
  a.split = p.split;
  a.chunk = p.chunk;
  a.part = static_cast<float*>(workspace);
  return launch_status(launch_attention(dtype, a, static_cast<hipStream_t>(stream)));
}

size_t w4a16_attention_backward_workspace_bytes(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D,
                                                int64_t window) {
  if (Tq <= 0 || bad_group(Hq, Hk) || bad_attn_dim(D) || window < 0) return 0;
  const size_t part = std::max(attn_split(kAttnDq, B, Tq, Tk, Hq, Hk, D, window).floats,
                               attn_split(kAttnDkv, B, Tq, Tk, Hq, Hk, D, window).floats);
  return (delta_floats(Tq, Hq) + part) * sizeof(float);
}

int w4a16_attention_backward(const void* dout, const void* q, int64_t q_token, int64_t q_head, const void* k,
                             int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                             const void* out, const float* lse, const int32_t* cu_q, const int32_t* cu_k, void* dq,
                             void* dk, void* dv, int dtype, int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk,
                             int64_t D, float scale, int causal, int64_t window, void* workspace,
                             size_t workspace_bytes, void* stream) {
  AttnArgs a;
  const int st = attn_args(a, {q, q_token, q_head}, {k, k_token, k_head}, {v, v_token, v_head}, cu_q, cu_k, dtype, B,
                           Tq, Tk, Hq, Hk, D, scale, causal, window);
  if (st != W4A16_OK) return st;
  if ((dk == nullptr) != (dv == nullptr)) return W4A16_ERR_NULL;
  if (Tq > 0 && (!dout || !out || !lse)) return W4A16_ERR_NULL;
  const void* p[] = {dout, out, dq, dk, dv, workspace};
  for (const void* x : p)
    if (!aligned16(x)) return W4A16_ERR_ALIGN;
  if (Tq > 0 && (workspace == nullptr ||
                 workspace_bytes < w4a16_attention_backward_workspace_bytes(B, Tq, Tk, Hq, Hk, D, window)))
    return W4A16_ERR_WORKSPACE;
  a.dout = dout;
  a.out = const_cast<void*>(out);
  a.lse = const_cast<float*>(lse);
  a.delta = static_cast<float*>(workspace);
  a.part = Tq > 0 ? a.delta + delta_floats(Tq, Hq) : nullptr;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  return launch_status(launch_attention_backward(dtype, a, static_cast<hipStream_t>(stream)));
}

size_t w4a16_decode_attention_workspace_bytes(int64_t B, int64_t Hq, int64_t Hk, int64_t D, int64_t keys) {
  if (B <= 0 || bad_group(Hq, Hk) || bad_attn_dim(D) || keys <= 0) return 0;
  if (decode_attn_whole(D, keys)) return 0;
  return decode_attn_part_floats(decode_attn_groups(B, Hq, Hk, D, keys), D) * sizeof(float);
}

int w4a16_decode_attention(const void* q, int64_t q_token, int64_t q_head, const void* k_cache, int64_t k_page_stride,
                           const void* v_cache, int64_t v_page_stride, const int32_t* block_table,
                           const int32_t* lengths, void* out, int dtype, int64_t B, int64_t Hq, int64_t Hk, int64_t D,
                           int64_t pages, int64_t page_size, int64_t width, float scale, int64_t window,
                           void* workspace, size_t workspace_bytes, void* stream) {
  const Heads h{q, q_token, q_head};
  if ((dtype != W4A16_BF16 && dtype != W4A16_F16) || B < 0 || B > kMaxSequences || bad_group(Hq, Hk) ||
      bad_attn_dim(D) || bad_page(page_size) || pages <= 0 || pages * page_size > INT32_MAX || width <= 0 ||
      width * page_size > INT32_MAX - 256 || bad_scale(scale) || window < 0 || bad_stride(h, 2) ||
      k_page_stride < Hk * page_size * D || v_page_stride < Hk * page_size * D)
    return W4A16_ERR_SHAPE;
  const int64_t units = B * Hk * ((Hq / Hk + 15) / 16), keys = width * page_size;
  if (units > kMaxBlocks || units * ((keys + 127) / 128 + 1) > INT32_MAX) return W4A16_ERR_SHAPE;
  if (B == 0) return W4A16_OK;
  if (!q || !k_cache || !v_cache || !block_table || !lengths || !out) return W4A16_ERR_NULL;
  if (odd(h, 2) || !aligned16(k_cache) || !aligned16(v_cache) || k_page_stride % 8 != 0 || v_page_stride % 8 != 0 ||
      !aligned16(out) || !aligned16(workspace))
    return W4A16_ERR_ALIGN;
  const size_t need = w4a16_decode_attention_workspace_bytes(B, Hq, Hk, D, keys);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return W4A16_ERR_WORKSPACE;
  DecodeAttnArgs a{};
  a.q = q;
  a.q_stride = 2 * q_token;
  a.q_head = 2 * q_head;
  a.kc = k_cache;
  a.vc = v_cache;
  a.k_page = 2 * k_page_stride;
  a.v_page = 2 * v_page_stride;
  a.out = out;
  a.table = block_table;
  a.lengths = lengths;
  a.part = static_cast<float*>(workspace);
  a.B = (int)B;
  a.Hq = (int)Hq;
  a.Hk = (int)Hk;
  a.group = (int)(Hq / Hk);
  a.D = (int)D;
  a.page_log2 = log2_of(page_size);
  a.pages = (int)pages;
  a.width = (int)width;
  a.scale2 = scale * 1.4426950408889634f;
  a.window = (int)std::min<int64_t>(window, INT32_MAX);
  a.groups = decode_attn_groups(B, Hq, Hk, D, keys);
  a.whole = decode_attn_whole(D, keys);
  return launch_status(launch_decode_attention(dtype, a, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
