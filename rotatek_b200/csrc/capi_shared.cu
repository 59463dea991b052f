// extern "C" entry points for serving many questions on shared prefixes
// (declared in include/rotatek_b200.h): rtk_shared_decode, rtk_append_text,
// rtk_read_text, rtk_verify_drafts.  Validation, kernel choice and launches;
// nothing allocates device memory or synchronises the stream.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <initializer_list>

#include "../../include/rotatek_b200.h"
#include "decode.h"
#include "shared.h"

namespace rtk {
bool encode_rows_map(CUtensorMap *map, const rtk_tensor *t, int box_inner, int box_rows);   // capi.cu
}

namespace {

int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return rtk::report_error(code, buf);
}

int cuda_fail(cudaError_t e, const char *what) { return fail(RTK_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e)); }

// `t` has these dimensions (-1: any)
bool dims(const rtk_tensor *t, std::initializer_list<int64_t> want) {
  if (t == nullptr || t->ndim != (int)want.size()) return false;
  int i = 0;
  for (int64_t w : want) {
    if (w >= 0 && t->shape[i] != w) return false;
    if (t->shape[i] < 0) return false;
    ++i;
  }
  return true;
}

bool float_type(int dt) { return dt == RTK_F32 || dt == RTK_BF16 || dt == RTK_F16; }

rtk::SharedTensor view(const rtk_tensor *t) {
  rtk::SharedTensor v;
  std::memset(&v, 0, sizeof(v));
  if (t != nullptr) {
    v.data = t->data;
    for (int i = 0; i < t->ndim; ++i) v.s[i] = t->stride[i];
  }
  return v;
}

// a tensor that a kernel reads or writes has an address unless it is empty (or not given)
bool present(const rtk_tensor *t) {
  if (t == nullptr) return true;
  int64_t n = 1;
  for (int i = 0; i < t->ndim; ++i) n *= t->shape[i];
  return n == 0 || t->data != nullptr;
}

constexpr int64_t kMaxInt = (1ll << 31) - 1;

// Rows (the last dimension) that 16-byte accesses can take: unit stride, an aligned
// address and strides of whole 16 bytes wherever a dimension has more than one entry.
bool rows16(const rtk_tensor *t, int esize) {
  const int n = t->ndim;
  if (t->shape[n - 1] > 1 && t->stride[n - 1] != 1) return false;
  if (reinterpret_cast<uintptr_t>(t->data) % 16 != 0) return false;
  for (int i = 0; i + 1 < n; ++i)
    if (t->shape[i] > 1 && (t->stride[i] * esize) % 16 != 0) return false;
  return true;
}

// ---- workspace of the tensor-core path: the prefix partials, the text's
struct SharedSpace {
  size_t prefix_ml, prefix_acc, text_ml, text_acc, bytes;
};

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

SharedSpace shared_space(const rtk::PrefixSplit &sp, int64_t batch, int64_t kv_heads, int64_t rows, int64_t chunks) {
  SharedSpace w;
  const size_t slots = (size_t)sp.slots() * 128, text = (size_t)(batch * kv_heads * chunks * rows);
  w.prefix_ml = 0;
  w.prefix_acc = up256(w.prefix_ml + slots * 8);
  w.text_ml = up256(w.prefix_acc + slots * 512);
  w.text_acc = up256(w.text_ml + text * 8);
  w.bytes = up256(w.text_acc + text * 512);
  return w;
}

int64_t text_chunks(int64_t batch, int64_t kv_heads, int64_t rows, int64_t cap) {
  const int64_t chunk = rtk::text_chunk(batch, kv_heads, rows, cap);
  return (cap + chunk - 1) / chunk;
}

int current_device() {
  int d = 0;
  cudaGetDevice(&d);
  return d;
}

}  // namespace

extern "C" {

size_t rtk_shared_decode_workspace_size(int64_t prefixes, int64_t batch, int64_t tokens, int64_t q_heads,
                                        int64_t kv_heads, int64_t seq_full, int64_t seq_sparse, int64_t text_cap,
                                        int32_t device) {
  if (prefixes < 1 || kv_heads < 1 || batch < 0 || tokens < 0) return 0;
  const int64_t groups = q_heads / kv_heads;
  const rtk::PrefixSplit sp =
      rtk::prefix_split(prefixes, batch / prefixes, tokens, groups, kv_heads, seq_full, seq_sparse, text_cap,
                        rtk::device_sms(device));
  return shared_space(sp, batch, kv_heads, tokens * groups, text_chunks(batch, kv_heads, tokens * groups, text_cap)).bytes;
}

int rtk_shared_decode(const rtk_tensor *q, const rtk_tensor *R_partial, const rtk_tensor *delta_mu,
                      const rtk_tensor *k_full, const rtk_tensor *v_full, const rtk_tensor *mask_full,
                      const rtk_tensor *k_sparse, const rtk_tensor *v_sparse, const rtk_tensor *k_text,
                      const rtk_tensor *v_text, const rtk_tensor *k_scale, const rtk_tensor *v_scale,
                      const rtk_tensor *text_lens, int64_t num_kv_groups, const rtk_tensor *out, void *workspace,
                      size_t workspace_bytes, void *status, void *stream) {
  rtk::report_error(RTK_OK, "");
  if (!dims(q, {-1, -1, -1, -1})) return fail(RTK_ERR_INVALID, "q must be [B, T, H_q, D]");
  if (!dims(R_partial, {-1, -1, -1, -1})) return fail(RTK_ERR_INVALID, "R_partial must be [P, H_kv, D, D_keep]");
  const int64_t B = q->shape[0], T = q->shape[1], Hq = q->shape[2], D = q->shape[3];
  const int64_t P = R_partial->shape[0], Hkv = R_partial->shape[1], DK = R_partial->shape[3];
  if (P < 1 || B % P != 0)
    return fail(RTK_ERR_INVALID, "B=%lld questions are not the same number for each of P=%lld prefixes", (long long)B,
                (long long)P);
  if (num_kv_groups <= 0 || Hq != Hkv * num_kv_groups)
    return fail(RTK_ERR_INVALID, "H_q=%lld is not H_kv=%lld * num_kv_groups=%lld", (long long)Hq, (long long)Hkv,
                (long long)num_kv_groups);
  if (!float_type(q->dtype)) return fail(RTK_ERR_INVALID, "q dtype must be float32, bfloat16 or float16");
  if (D < 1 || !dims(R_partial, {P, Hkv, D, -1}) || DK < 1 || DK > D)
    return fail(RTK_ERR_INVALID, "R_partial must be [P, H_kv, D, D_keep] with 1 <= D_keep <= D");
  if (delta_mu != nullptr && !dims(delta_mu, {P, Hkv, D})) return fail(RTK_ERR_INVALID, "delta_mu must be [P, H_kv, D]");
  if (!dims(k_full, {P, Hkv, -1, D})) return fail(RTK_ERR_INVALID, "k_full must be [P, H_kv, S_full, D]");
  const int64_t Sf = k_full->shape[2];
  if (!dims(v_full, {P, Hkv, Sf, D})) return fail(RTK_ERR_INVALID, "v_full must be [P, H_kv, S_full, D]");
  if (mask_full != nullptr && (!dims(mask_full, {P, Sf}) || mask_full->dtype != RTK_U8))
    return fail(RTK_ERR_INVALID, "mask_full must be a uint8 [P, S_full]");
  if (!dims(k_sparse, {P, Hkv, -1, DK})) return fail(RTK_ERR_INVALID, "k_sparse must be [P, H_kv, S_sparse, D_keep]");
  const int64_t Sv = k_sparse->shape[2];
  if (!dims(v_sparse, {P, Hkv, Sv, D})) return fail(RTK_ERR_INVALID, "v_sparse must be [P, H_kv, S_sparse, D]");
  if (!dims(k_text, {B, Hkv, -1, D})) return fail(RTK_ERR_INVALID, "k_text must be [B, H_kv, C, D]");
  const int64_t C = k_text->shape[2];
  if (!dims(v_text, {B, Hkv, C, D})) return fail(RTK_ERR_INVALID, "v_text must be [B, H_kv, C, D]");
  const bool fp8 = k_scale != nullptr || v_scale != nullptr;
  if (fp8) {
    if (k_text->dtype != RTK_U8 || v_text->dtype != RTK_U8)
      return fail(RTK_ERR_INVALID, "k_text and v_text must be uint8 (e4m3) where scales are given");
    for (const rtk_tensor *t : {k_scale, v_scale})
      if (t == nullptr || !dims(t, {B, Hkv, C}) || t->dtype != RTK_F32)
        return fail(RTK_ERR_INVALID, "k_scale and v_scale must both be float32 [B, H_kv, C]");
  } else if (k_text->dtype != q->dtype || v_text->dtype != q->dtype) {
    return fail(RTK_ERR_INVALID, "k_text and v_text must have q's dtype, or be e4m3 with k_scale and v_scale");
  }
  if (!dims(text_lens, {B}) || text_lens->dtype != RTK_I32) return fail(RTK_ERR_INVALID, "text_lens must be an int32 [B]");
  if (!dims(out, {B, T, Hq, D}) || out->dtype != q->dtype)
    return fail(RTK_ERR_INVALID, "out must be [B, T, H_q, D] in q's dtype");
  for (const rtk_tensor *t : {R_partial, k_full, v_full, k_sparse, v_sparse})
    if (t->dtype != q->dtype)
      return fail(RTK_ERR_INVALID, "q, R_partial, delta_mu, k_full, v_full, k_sparse and v_sparse must share a dtype");
  if (delta_mu != nullptr && delta_mu->dtype != q->dtype)
    return fail(RTK_ERR_INVALID, "q, R_partial, delta_mu, k_full, v_full, k_sparse and v_sparse must share a dtype");
  if (D > 256) return fail(RTK_ERR_UNSUPPORTED, "head_dim %lld > 256 is not supported", (long long)D);
  if (B * T * Hq > kMaxInt || Sf > kMaxInt || Sv > kMaxInt || C > kMaxInt)
    return fail(RTK_ERR_UNSUPPORTED, "more than 2^31 - 1 query rows or tokens");
  if (B * T * Hq == 0) return RTK_OK;
  for (const rtk_tensor *t : {q, R_partial, delta_mu, k_full, v_full, mask_full, k_sparse, v_sparse, k_text, v_text,
                              k_scale, v_scale, text_lens, out})
    if (!present(t)) return fail(RTK_ERR_INVALID, "a tensor that is not empty has no address");

  rtk::SharedParams p;
  std::memset(&p, 0, sizeof(p));
  p.dtype = q->dtype;
  p.text_fp8 = fp8;
  p.prefixes = (int)P; p.questions = (int)(B / P); p.tokens = (int)T;
  p.q_heads = (int)Hq; p.kv_heads = (int)Hkv; p.groups = (int)num_kv_groups;
  p.head_dim = (int)D; p.head_dim_keep = (int)DK;
  p.seq_full = (int)Sf; p.seq_sparse = (int)Sv; p.cap = (int)C;
  p.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)D));
  p.q = view(q); p.R = view(R_partial); p.dm = view(delta_mu);
  p.kf = view(k_full); p.vf = view(v_full); p.mask = view(mask_full);
  p.ks = view(k_sparse); p.vs = view(v_sparse);
  p.kt = view(k_text); p.vt = view(v_text); p.ksc = view(k_scale); p.vsc = view(v_scale);
  p.lens = static_cast<const int *>(text_lens->data); p.lens_s = text_lens->stride[0];
  p.out = out->data;
  for (int i = 0; i < 4; ++i) p.o_s[i] = out->stride[i];
  const cudaStream_t st = static_cast<cudaStream_t>(stream);

  // ---- tensor-core path
  bool tc = (q->dtype == RTK_BF16 || q->dtype == RTK_F16) && D == 128 && rows16(q, 2) && (C == 0 || (rows16(k_text, fp8 ? 1 : 2) && rows16(v_text, fp8 ? 1 : 2)));
  if (Sv > 0)
    tc = tc && (DK == 16 || DK == 32 || DK == 64) && (delta_mu == nullptr || delta_mu->stride[2] == 1);
  rtk::PrefixMaps maps;
  std::memset(&maps, 0, sizeof(maps));
  if (tc && Sf > 0) tc = rtk::encode_rows_map(&maps.kf, k_full, 64, 64) && rtk::encode_rows_map(&maps.vf, v_full, 64, 64);
  if (tc && Sv > 0)
    tc = rtk::encode_rows_map(&maps.ks, k_sparse, (int)DK, 128) && rtk::encode_rows_map(&maps.vs, v_sparse, 64, 128);
  if (!tc) {
    const cudaError_t e = rtk::launch_shared_simt(p, st);
    if (e != cudaSuccess) return cuda_fail(e, "shared decode (generic kernel) launch");
    return RTK_OK;
  }
  const int device = current_device();
  const rtk::PrefixSplit sp =
      rtk::prefix_split(P, B / P, T, num_kv_groups, Hkv, Sf, Sv, C, rtk::device_sms(device));
  const int64_t rows = T * num_kv_groups, chunks = text_chunks(B, Hkv, rows, C);
  if ((int64_t)sp.rows != B / P * rows || (int64_t)P * Hkv * sp.row_tiles > kMaxInt / 256 || chunks > 65535 ||
      rows > 65535 * 16 || B * Hkv > kMaxInt)
    return fail(RTK_ERR_UNSUPPORTED, "too many query rows or text tokens");
  const SharedSpace w = shared_space(sp, B, Hkv, rows, chunks);
  if (workspace == nullptr || workspace_bytes < w.bytes)
    return fail(RTK_ERR_WORKSPACE, "workspace has %zu bytes, needs %zu", workspace == nullptr ? (size_t)0 : workspace_bytes,
                w.bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(RTK_ERR_INVALID, "workspace must be 16-byte aligned");
  unsigned char *ws = static_cast<unsigned char *>(workspace);
  if (Sv == 0) p.head_dim_keep = 16;               // no visual block uses it
  cudaError_t e = cudaSuccess;
  rtk::MergeParams mp;
  std::memset(&mp, 0, sizeof(mp));
  mp.s = p;
  mp.split = sp;
  mp.has_prefix = Sf + Sv > 0;
  mp.has_text = C > 0;
  mp.text_rows = (int)rows; mp.text_chunk = rtk::text_chunk(B, Hkv, rows, C); mp.text_chunks = (int)chunks;
  float *pml = reinterpret_cast<float *>(ws + w.prefix_ml), *pacc = reinterpret_cast<float *>(ws + w.prefix_acc);
  float *tml = reinterpret_cast<float *>(ws + w.text_ml), *tacc = reinterpret_cast<float *>(ws + w.text_acc);
  mp.prefix_ml = pml; mp.prefix_acc = pacc; mp.text_ml = tml; mp.text_acc = tacc;
  if (mp.has_prefix) {
    rtk::PrefixParams pp;
    pp.s = p;
    pp.split = sp;
    rtk_tensor Rt = *R_partial;                      // its columns as rows
    std::swap(Rt.shape[2], Rt.shape[3]);
    std::swap(Rt.stride[2], Rt.stride[3]);
    pp.R_layout = rows16(R_partial, 2) ? 1 : rows16(&Rt, 2) ? 2 : 0;
    pp.ml = pml; pp.acc = pacc;
    pp.status = static_cast<unsigned int *>(status);
    e = rtk::launch_shared_prefix(maps, pp, st);
    if (e != cudaSuccess) return cuda_fail(e, "shared decode (prefix kernel) launch");
  }
  if (mp.has_text) {
    rtk::TextParams tp;
    tp.s = p;
    tp.rows = (int)rows; tp.chunk = mp.text_chunk; tp.chunks = (int)chunks;
    tp.beside = mp.has_prefix;
    tp.ml = tml; tp.acc = tacc;
    e = rtk::launch_shared_text(tp, st);
    if (e != cudaSuccess) return cuda_fail(e, "shared decode (text kernel) launch");
  }
  e = rtk::launch_shared_merge(mp, st);
  if (e != cudaSuccess) return cuda_fail(e, "shared decode (merge kernel) launch");
  return RTK_OK;
}

int rtk_read_shared_status(void *stream, uint32_t *status) {
  rtk::report_error(RTK_OK, "");
  void *word = nullptr;
  const cudaError_t e = rtk::shared_status_address(&word);
  if (e != cudaSuccess) return cuda_fail(e, "rtk_read_shared_status");
  return rtk_read_status(word, stream, status);
}

int rtk_append_text(const rtk_tensor *k_new, const rtk_tensor *v_new, const rtk_tensor *text_lens,
                    const rtk_tensor *counts, const rtk_tensor *k_text, const rtk_tensor *v_text,
                    const rtk_tensor *k_scale, const rtk_tensor *v_scale, void *stream) {
  rtk::report_error(RTK_OK, "");
  if (!dims(k_new, {-1, -1, -1, -1})) return fail(RTK_ERR_INVALID, "k_new must be [B, H_kv, T, D]");
  const int64_t B = k_new->shape[0], H = k_new->shape[1], T = k_new->shape[2], D = k_new->shape[3];
  if (!dims(v_new, {B, H, T, D})) return fail(RTK_ERR_INVALID, "v_new must be [B, H_kv, T, D]");
  if (!dims(k_text, {B, H, -1, D})) return fail(RTK_ERR_INVALID, "k_text must be [B, H_kv, C, D]");
  const int64_t C = k_text->shape[2];
  if (!dims(v_text, {B, H, C, D})) return fail(RTK_ERR_INVALID, "v_text must be [B, H_kv, C, D]");
  if (!float_type(k_new->dtype) || v_new->dtype != k_new->dtype)
    return fail(RTK_ERR_INVALID, "k_new and v_new must both be float32, bfloat16 or float16");
  const bool fp8 = k_scale != nullptr || v_scale != nullptr;
  if (fp8) {
    if (k_text->dtype != RTK_U8 || v_text->dtype != RTK_U8)
      return fail(RTK_ERR_INVALID, "k_text and v_text must be uint8 (e4m3) where scales are given");
    for (const rtk_tensor *t : {k_scale, v_scale})
      if (t == nullptr || !dims(t, {B, H, C}) || t->dtype != RTK_F32)
        return fail(RTK_ERR_INVALID, "k_scale and v_scale must both be float32 [B, H_kv, C]");
  } else if (k_text->dtype != k_new->dtype || v_text->dtype != k_new->dtype) {
    return fail(RTK_ERR_INVALID, "k_text and v_text must have k_new's dtype, or be e4m3 with k_scale and v_scale");
  }
  if (!dims(text_lens, {B}) || text_lens->dtype != RTK_I32) return fail(RTK_ERR_INVALID, "text_lens must be an int32 [B]");
  if (counts != nullptr && (!dims(counts, {B}) || counts->dtype != RTK_I32))
    return fail(RTK_ERR_INVALID, "counts must be an int32 [B]");
  if (2 * B * H * T > kMaxInt || C > kMaxInt) return fail(RTK_ERR_UNSUPPORTED, "more than 2^31 - 1 rows");
  if (B * H * T * D == 0 || C == 0) return RTK_OK;
  for (const rtk_tensor *t : {k_new, v_new, k_text, v_text, k_scale, v_scale, text_lens, counts})
    if (!present(t)) return fail(RTK_ERR_INVALID, "a tensor that is not empty has no address");

  rtk::AppendParams p;
  std::memset(&p, 0, sizeof(p));
  p.dtype = k_new->dtype; p.quantize = fp8;
  p.batch = (int)B; p.heads = (int)H; p.tokens = (int)T; p.cap = (int)C; p.head_dim = (int)D;
  p.src[0] = view(k_new); p.src[1] = view(v_new);
  p.dst[0] = view(k_text); p.dst[1] = view(v_text);
  p.scale[0] = view(k_scale); p.scale[1] = view(v_scale);
  p.lens = static_cast<const int *>(text_lens->data); p.lens_s = text_lens->stride[0];
  if (counts != nullptr) { p.counts = static_cast<const int *>(counts->data); p.counts_s = counts->stride[0]; }
  const cudaError_t e = rtk::launch_append_text(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "text append launch");
  return RTK_OK;
}

int rtk_read_text(const rtk_tensor *k_text, const rtk_tensor *v_text, const rtk_tensor *k_scale,
                  const rtk_tensor *v_scale, const rtk_tensor *text_lens, const rtk_tensor *k_out,
                  const rtk_tensor *v_out, void *stream) {
  rtk::report_error(RTK_OK, "");
  if (!dims(k_text, {-1, -1, -1, -1}) || k_text->dtype != RTK_U8)
    return fail(RTK_ERR_INVALID, "k_text must be a uint8 (e4m3) [B, H_kv, C, D]");
  const int64_t B = k_text->shape[0], H = k_text->shape[1], C = k_text->shape[2], D = k_text->shape[3];
  if (!dims(v_text, {B, H, C, D}) || v_text->dtype != RTK_U8)
    return fail(RTK_ERR_INVALID, "v_text must be a uint8 (e4m3) [B, H_kv, C, D]");
  for (const rtk_tensor *t : {k_scale, v_scale})
    if (!dims(t, {B, H, C}) || t->dtype != RTK_F32)
      return fail(RTK_ERR_INVALID, "k_scale and v_scale must both be float32 [B, H_kv, C]");
  if (!dims(text_lens, {B}) || text_lens->dtype != RTK_I32) return fail(RTK_ERR_INVALID, "text_lens must be an int32 [B]");
  for (const rtk_tensor *t : {k_out, v_out})
    if (!dims(t, {B, H, C, D}) || !float_type(t->dtype) || t->dtype != k_out->dtype)
      return fail(RTK_ERR_INVALID, "k_out and v_out must be [B, H_kv, C, D], both float32, bfloat16 or float16");
  if (2 * B * H * C > kMaxInt) return fail(RTK_ERR_UNSUPPORTED, "more than 2^31 - 1 rows");
  if (B * H * C * D == 0) return RTK_OK;
  for (const rtk_tensor *t : {k_text, v_text, k_scale, v_scale, text_lens, k_out, v_out})
    if (!present(t)) return fail(RTK_ERR_INVALID, "a tensor that is not empty has no address");

  rtk::ReadParams p;
  std::memset(&p, 0, sizeof(p));
  p.dtype = k_out->dtype;
  p.batch = (int)B; p.heads = (int)H; p.cap = (int)C; p.head_dim = (int)D;
  p.src[0] = view(k_text); p.src[1] = view(v_text);
  p.scale[0] = view(k_scale); p.scale[1] = view(v_scale);
  p.dst[0] = view(k_out); p.dst[1] = view(v_out);
  p.lens = static_cast<const int *>(text_lens->data); p.lens_s = text_lens->stride[0];
  const cudaError_t e = rtk::launch_read_text(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "text read launch");
  return RTK_OK;
}

size_t rtk_verify_drafts_workspace_size(int64_t batch, int64_t drafts, int64_t vocab) {
  if (batch < 0 || drafts < 0 || vocab < 0) return 0;
  return rtk::verify_workspace_bytes(batch, drafts, vocab);
}

int rtk_verify_drafts(const rtk_tensor *target_logits, const rtk_tensor *draft_tokens, const rtk_tensor *draft_logits,
                      const rtk_tensor *uniforms, const rtk_tensor *noise, const rtk_tensor *temperature,
                      const rtk_tensor *draft_lens, const rtk_tensor *tokens_out, const rtk_tensor *accepted_out,
                      void *workspace, size_t workspace_bytes, void *stream) {
  rtk::report_error(RTK_OK, "");
  if (!dims(target_logits, {-1, -1, -1}) || target_logits->shape[1] < 1 || target_logits->shape[2] < 1)
    return fail(RTK_ERR_INVALID, "target_logits must be [B, T + 1, V]");
  const int64_t B = target_logits->shape[0], T = target_logits->shape[1] - 1, V = target_logits->shape[2];
  if (!float_type(target_logits->dtype))
    return fail(RTK_ERR_INVALID, "target_logits dtype must be float32, bfloat16 or float16");
  if (!dims(draft_tokens, {B, T}) || draft_tokens->dtype != RTK_I64)
    return fail(RTK_ERR_INVALID, "draft_tokens must be an int64 [B, T]");
  if (draft_logits != nullptr && (!dims(draft_logits, {B, T, V}) || draft_logits->dtype != target_logits->dtype))
    return fail(RTK_ERR_INVALID, "draft_logits must be [B, T, V] in target_logits' dtype");
  if (!dims(uniforms, {B, T}) || uniforms->dtype != RTK_F32) return fail(RTK_ERR_INVALID, "uniforms must be a float32 [B, T]");
  if (!dims(noise, {B, V}) || noise->dtype != RTK_F32) return fail(RTK_ERR_INVALID, "noise must be a float32 [B, V]");
  if (!dims(temperature, {B}) || temperature->dtype != RTK_F32)
    return fail(RTK_ERR_INVALID, "temperature must be a float32 [B]");
  if (draft_lens != nullptr && (!dims(draft_lens, {B}) || draft_lens->dtype != RTK_I32))
    return fail(RTK_ERR_INVALID, "draft_lens must be an int32 [B]");
  if (!dims(tokens_out, {B, T + 1}) || tokens_out->dtype != RTK_I64 || (B > 1 && tokens_out->stride[0] != T + 1) ||
      (T > 0 && tokens_out->stride[1] != 1))
    return fail(RTK_ERR_INVALID, "tokens_out must be a contiguous int64 [B, T + 1]");
  if (!dims(accepted_out, {B}) || accepted_out->dtype != RTK_I32 || (B > 1 && accepted_out->stride[0] != 1))
    return fail(RTK_ERR_INVALID, "accepted_out must be a contiguous int32 [B]");
  if (V > 1 && (target_logits->stride[2] != 1 || noise->stride[1] != 1 ||
                (draft_logits != nullptr && draft_logits->stride[2] != 1)))
    return fail(RTK_ERR_UNSUPPORTED, "logits and noise need a unit vocabulary stride");
  if (T > 64) return fail(RTK_ERR_UNSUPPORTED, "at most 64 drafted tokens (got %lld)", (long long)T);
  if (B > 65535 || V > (1 << 30)) return fail(RTK_ERR_UNSUPPORTED, "at most 65535 questions and a vocabulary of 2^30");
  if (B == 0) return RTK_OK;
  for (const rtk_tensor *t : {target_logits, draft_tokens, draft_logits, uniforms, noise, temperature, draft_lens,
                              tokens_out, accepted_out})
    if (!present(t)) return fail(RTK_ERR_INVALID, "a tensor that is not empty has no address");
  const size_t need = rtk::verify_workspace_bytes(B, T, V);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(RTK_ERR_WORKSPACE, "workspace has %zu bytes, needs %zu", workspace == nullptr ? (size_t)0 : workspace_bytes, need);
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(RTK_ERR_INVALID, "workspace must be 16-byte aligned");

  rtk::VerifyParams p;
  std::memset(&p, 0, sizeof(p));
  p.dtype = target_logits->dtype;
  p.batch = (int)B; p.drafts = (int)T; p.vocab = (int)V;
  p.target = view(target_logits); p.draft = view(T > 0 ? draft_logits : nullptr);
  p.tokens = static_cast<const long long *>(draft_tokens->data);
  p.uniforms = static_cast<const float *>(uniforms->data);
  for (int i = 0; i < 2; ++i) { p.tok_s[i] = draft_tokens->stride[i]; p.uni_s[i] = uniforms->stride[i]; }
  p.noise = static_cast<const float *>(noise->data); p.noise_s = noise->stride[0];
  p.temperature = static_cast<const float *>(temperature->data); p.temp_s = temperature->stride[0];
  if (draft_lens != nullptr) { p.draft_lens = static_cast<const int *>(draft_lens->data); p.dl_s = draft_lens->stride[0]; }
  p.out_tokens = static_cast<long long *>(tokens_out->data);
  p.accepted = static_cast<int *>(accepted_out->data);
  p.workspace = workspace;
  const cudaError_t e = rtk::launch_verify(p, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "draft verification launch");
  return RTK_OK;
}

}  // extern "C"
