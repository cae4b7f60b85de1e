// C entries of differential attention: argument checks and the dispatch by element type (kernels: diff_attn.inl).
#include "diff_attn.h"

namespace ubv {
int diff_attn_forward_f32(const DiffAttnArgs&, void*, int64_t, hipStream_t);
int diff_attn_forward_f16(const DiffAttnArgs&, void*, int64_t, hipStream_t);
int diff_attn_forward_bf16(const DiffAttnArgs&, void*, int64_t, hipStream_t);
int diff_attn_backward_f32(const DiffAttnArgs&, float*, int64_t, hipStream_t);
int diff_attn_backward_f16(const DiffAttnArgs&, float*, int64_t, hipStream_t);
int diff_attn_backward_bf16(const DiffAttnArgs&, float*, int64_t, hipStream_t);
int64_t diff_attn_bytes_f32(const DiffAttnArgs&, bool);
int64_t diff_attn_bytes_f16(const DiffAttnArgs&, bool);
int64_t diff_attn_bytes_bf16(const DiffAttnArgs&, bool);

// rows of a group, keys and heads count in 32 bits, the next tile's included
static bool attn_in_reach(int B, int H, int Hk, int Nq, int Nk, int causal) {
  constexpr int64_t most = (int64_t(1) << 31) - 256;
  return (int64_t)(H / Hk) * Nq < most && Nk < most && (int64_t)B * H < (int64_t(1) << 31) && (!causal || (int64_t)Nq + Nk < (int64_t(1) << 31));
}
static int64_t attn_part_bytes(int B, int H, int Hk, int Nq, int Nk, int Dh, int Dv, int causal, int dtype, bool backward) {
  if (B <= 0 || Hk <= 0 || H < Hk || H % Hk != 0 || Nq <= 0 || Nk <= 0 || Dh <= 0 || Dv <= 0 || Dh > 128 || Dv > 256) return 0;
  if (!attn_in_reach(B, H, Hk, Nq, Nk, causal)) return 0;      // (such a call is refused)
  DiffAttnArgs a{};
  a.B = B; a.H = H; a.Hk = Hk; a.G = H / Hk; a.Nq = Nq; a.Nk = Nk; a.Dh = Dh; a.Dv = Dv; a.R = a.G * Nq; a.causal = causal != 0;
  return dtype == UBV_F32 ? diff_attn_bytes_f32(a, backward) : dtype == UBV_F16 ? diff_attn_bytes_f16(a, backward) : diff_attn_bytes_bf16(a, backward);
}
// the backward pass's rows: statistics (float4 + float2) and grad_lam's part, then the splits' sums
static int64_t attn_row_bytes(int64_t rows) { return (28 * rows + 15) / 16 * 16; }

// what forward and backward share: shapes, strides (in elements: q 4, k 4, v 3, grad_out 3, mask 4), masks, dropout
static int attn_args(DiffAttnArgs& a, const void* q, const void* k, const void* v, const float* lam, const uint8_t* kpm,
                     const void* mask, int mask_kind, const int64_t* strides, int B, int H, int Hk, int Nq, int Nk, int Dh, int Dv,
                     float scale, int causal, float p, uint64_t seed, const uint64_t* seed_dev, int dtype, const char* who) {
  UBV_CHECK_ARG(q && k && v && lam && strides, "%s: null pointer", who);
  UBV_CHECK_ARG(dtype >= 0 && dtype <= 2, "%s: unknown dtype %d", who, dtype);
  UBV_CHECK_ARG(B > 0 && H > 0 && Hk > 0 && Nq > 0 && Nk > 0, "%s: empty shape B=%d H=%d Hk=%d Nq=%d Nk=%d", who, B, H, Hk, Nq, Nk);
  UBV_CHECK_ARG(H % Hk == 0, "%s: %d query heads do not share %d key heads evenly", who, H, Hk);
  UBV_CHECK_ARG(Dh > 0 && Dh <= 128 && Dv > 0 && Dv <= 256, "%s: head widths %d (at most 128) and %d (at most 256)", who, Dh, Dv);
  UBV_CHECK_ARG(attn_in_reach(B, H, Hk, Nq, Nk, causal), "%s: Nq=%d x %d heads, Nk=%d or B=%d x H=%d out of range", who, Nq, H / Hk, Nk, B, H);
  UBV_CHECK_ARG(p >= 0.0f && p <= 1.0f, "%s: p = %g must be in [0, 1]", who, (double)p);
  UBV_CHECK_ARG(scale >= 0.99e-30f && scale < 1.01e30f, "%s: scale %g must be in [1e-30, 1e30)", who, (double)scale);
  UBV_CHECK_ARG(mask_kind >= 0 && mask_kind <= 2 && (mask_kind == 0) == (mask == nullptr), "%s: mask kind %d", who, mask_kind);
  const int vec = dtype == UBV_F32 ? 4 : 8;
  for (int n = 0; n < 14; ++n)
    UBV_CHECK_ARG(strides[n] % vec == 0, "%s: stride %ld is no multiple of 16 bytes", who, (long)strides[n]);
  const int size = 16 / vec;                 // a staged tile is reached with 32-bit offsets from its first row
  for (int n : {1, 5, 9, 12})
    UBV_CHECK_ARG(strides[n] >= 0 && strides[n] * size < (1 << 24), "%s: token stride %ld is negative or over 16 MiB", who, (long)strides[n]);
  for (int n : {3, 7})
    UBV_CHECK_ARG(strides[n] >= 0 && strides[n] * size < (1 << 28), "%s: map stride %ld is negative or over 256 MiB", who, (long)strides[n]);
  UBV_CHECK_ARG(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 == 0, "%s: operands must be 16-byte aligned", who);
  a = DiffAttnArgs{};
  a.q = q; a.k = k; a.v = v; a.lam = lam; a.kpm = kpm; a.mask = mask; a.mask_kind = mask_kind;
  for (int n = 0; n < 4; ++n) { a.qs[n] = strides[n]; a.ks[n] = strides[4 + n]; a.ms[n] = strides[14 + n]; }
  for (int n = 0; n < 3; ++n) { a.vs[n] = strides[8 + n]; a.gs[n] = strides[11 + n]; }
  a.B = B; a.H = H; a.Hk = Hk; a.G = H / Hk; a.Nq = Nq; a.Nk = Nk; a.Dh = Dh; a.Dv = Dv; a.R = a.G * Nq;
  a.scale = scale; a.causal = causal != 0; a.n4 = (Nk + 3) / 4;
  drop_params16(p, a.t16, a.up);
  a.seed = seed; a.seed_dev = seed_dev;
  return UBV_OK;
}
}  // namespace ubv

extern "C" int64_t ubv_diff_attention_forward_workspace(int B, int H, int Hk, int Nq, int Nk, int Dh, int Dv, int causal, int dtype) {
  return ubv::attn_part_bytes(B, H, Hk, Nq, Nk, Dh, Dv, causal, dtype, false);
}

extern "C" int ubv_diff_attention_forward(const void* q, const void* k, const void* v, const float* lam, const uint8_t* key_padding_mask,
                                          const void* mask, int mask_kind, void* out, float* stat, float* maps,
                                          const int64_t* strides, int B, int H, int Hk, int Nq, int Nk, int Dh, int Dv, float scale,
                                          int causal, float p, uint64_t seed, const uint64_t* seed_dev, int dtype, void* workspace,
                                          int64_t workspace_bytes, void* stream) {
  using namespace ubv;
  DiffAttnArgs a;
  const int rc = attn_args(a, q, k, v, lam, key_padding_mask, mask, mask_kind, strides, B, H, Hk, Nq, Nk, Dh, Dv, scale, causal, p, seed,
                           seed_dev, dtype, "diff_attention_forward");
  if (rc) return rc;
  UBV_CHECK_ARG(out && (uintptr_t)out % 16 == 0 && ((uintptr_t)maps | (uintptr_t)stat | (uintptr_t)workspace) % 16 == 0 &&
                    (stat == nullptr) == (maps == nullptr),
                "diff_attention_forward: out, or stat without maps");
  a.out = out; a.stat = (float4*)stat; a.o = maps;
  hipStream_t st = as_stream(stream);
  switch (dtype) {
    case UBV_F32: return diff_attn_forward_f32(a, workspace, workspace_bytes, st);
    case UBV_F16: return diff_attn_forward_f16(a, workspace, workspace_bytes, st);
    default: return diff_attn_forward_bf16(a, workspace, workspace_bytes, st);
  }
}

extern "C" int64_t ubv_diff_attention_backward_workspace(int B, int H, int Hk, int Nq, int Nk, int Dh, int Dv, int causal, int dtype) {
  if (B <= 0 || H <= 0 || Nq <= 0) return 0;
  return ubv::attn_row_bytes((int64_t)B * H * Nq) + ubv::attn_part_bytes(B, H, Hk, Nq, Nk, Dh, Dv, causal, dtype, true);
}

extern "C" int ubv_diff_attention_backward(const void* grad_out, const void* q, const void* k, const void* v, const float* lam,
                                           const uint8_t* key_padding_mask, const void* mask, int mask_kind, const float* stat,
                                           const float* maps, void* grad_q, void* grad_k, void* grad_v, float* grad_lam,
                                           const int64_t* strides, int B, int H, int Hk, int Nq, int Nk, int Dh, int Dv, float scale,
                                           int causal, float p, uint64_t seed, const uint64_t* seed_dev, int dtype, void* workspace,
                                           int64_t workspace_bytes, void* stream) {
  using namespace ubv;
  DiffAttnArgs a;
  const int rc = attn_args(a, q, k, v, lam, key_padding_mask, mask, mask_kind, strides, B, H, Hk, Nq, Nk, Dh, Dv, scale, causal, p, seed,
                           seed_dev, dtype, "diff_attention_backward");
  if (rc) return rc;
  UBV_CHECK_ARG(grad_out && stat && maps && ((uintptr_t)grad_out | (uintptr_t)stat) % 16 == 0, "diff_attention_backward: grad_out, stat or maps");
  UBV_CHECK_ARG((grad_k == nullptr) == (grad_v == nullptr), "diff_attention_backward: grad_k and grad_v come together");
  UBV_CHECK_ARG(((uintptr_t)grad_q | (uintptr_t)grad_k | (uintptr_t)grad_v) % 16 == 0, "diff_attention_backward: gradients must be 16-byte aligned");
  UBV_CHECK_ARG(workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= attn_row_bytes((int64_t)B * H * Nq),
                "diff_attention_backward: the workspace is too small (%ld bytes)", (long)workspace_bytes);
  const int64_t rows = (int64_t)B * H * Nq;
  a.go = grad_out; a.stat = (float4*)const_cast<float*>(stat); a.o = const_cast<float*>(maps);
  a.gq = grad_q; a.gk = grad_k; a.gv = grad_v;
  a.row = (float4*)workspace; a.rowl = (float2*)(a.row + rows); a.dlrow = (float*)(a.rowl + rows);
  const int64_t part = workspace_bytes - attn_row_bytes(rows);
  a.part = (float*)((char*)workspace + attn_row_bytes(rows));
  hipStream_t st = as_stream(stream);
  switch (dtype) {
    case UBV_F32: return diff_attn_backward_f32(a, grad_lam, part, st);
    case UBV_F16: return diff_attn_backward_f16(a, grad_lam, part, st);
    default: return diff_attn_backward_bf16(a, grad_lam, part, st);
  }
}
