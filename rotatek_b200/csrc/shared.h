// Parameters shared by the kernels that serve many questions on shared
// prefixes (attention, text caches, draft verification) and their launchers.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace rtk {

struct SharedTensor {
  const void *data;
  long long s[4];    // element strides
};

// Attention of T new tokens per question over the question's prefix and its own
// text.  Question b belongs to prefix b / questions.  Strides in elements.
struct SharedParams {
  int dtype;                              // rtk_dtype of q, R, K, V and out
  int text_fp8;                           // kt / vt are e4m3 bytes with scales
  int prefixes, questions, tokens;        // B = prefixes * questions
  int q_heads, kv_heads, groups, head_dim, head_dim_keep;
  int seq_full, seq_sparse, cap;          // prompt, visual, text capacity
  float scale_log2;                       // log2(e) / sqrt(head_dim)
  SharedTensor q;                         // [B, T, H_q, D]
  SharedTensor R;                         // [P, H_kv, D, D_keep]
  SharedTensor dm;                        // [P, H_kv, D], data nullable
  SharedTensor kf, vf;                    // [P, H_kv, S_f, D]
  SharedTensor mask;                      // [P, S_f] uint8, data nullable
  SharedTensor ks, vs;                    // [P, H_kv, S_v, D_keep], [P, H_kv, S_v, D]
  SharedTensor kt, vt;                    // [B, H_kv, C, D]
  SharedTensor ksc, vsc;                  // [B, H_kv, C] f32 (text_fp8)
  const int *lens; long long lens_s;      // [B]
  void *out; long long o_s[4];            // [B, T, H_q, D]
};

// Generic kernel (shared_simt.cu): any dtype, any strides, head_dim <= 256.
cudaError_t launch_shared_simt(const SharedParams &p, cudaStream_t stream);

// New Keys and Values written into text caches at their lengths (text_cache.cu).
struct AppendParams {
  int dtype;                              // rtk_dtype of the new rows
  int quantize;                           // e4m3 rows + scales, else rows copied
  int batch, heads, tokens, cap, head_dim;
  SharedTensor src[2];                    // new Keys, Values [B, H, T, D]
  SharedTensor dst[2];                    // caches [B, H, C, D]
  SharedTensor scale[2];                  // [B, H, C] f32 (quantize)
  const int *lens; long long lens_s;      // [B]
  const int *counts; long long counts_s;  // [B], nullable: T for every question
};
cudaError_t launch_append_text(const AppendParams &p, cudaStream_t stream);

// 8-bit caches back in a 16- or 32-bit type (text_cache.cu).
struct ReadParams {
  int dtype;                              // rtk_dtype of the outputs
  int batch, heads, cap, head_dim;
  SharedTensor src[2], scale[2], dst[2];  // [B, H, C, D] u8, [B, H, C] f32, [B, H, C, D]
  const int *lens; long long lens_s;
};
cudaError_t launch_read_text(const ReadParams &p, cudaStream_t stream);

// Verification of drafted tokens (verify.cu).
struct VerifyParams {
  int dtype;                              // rtk_dtype of both logits
  int batch, drafts, vocab;
  SharedTensor target;                    // [B, T + 1, V], vocabulary stride 1
  SharedTensor draft;                     // [B, T, V], vocabulary stride 1, data nullable
  const long long *tokens; long long tok_s[2];      // [B, T]
  const float *uniforms; long long uni_s[2];        // [B, T]
  const float *noise; long long noise_s;            // [B, V], vocabulary stride 1
  const float *temperature; long long temp_s;       // [B]
  const int *draft_lens; long long dl_s;            // [B], nullable
  long long *out_tokens;                  // [B, T + 1] contiguous
  int *accepted;                          // [B] contiguous
  void *workspace;
};
size_t verify_workspace_bytes(long long batch, long long drafts, long long vocab);
cudaError_t launch_verify(const VerifyParams &p, int sms, cudaStream_t stream);

}  // namespace rtk
