// Parameters shared by the kernels that serve many questions on shared
// prefixes (attention, text caches, draft verification) and their launchers.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace rtk {

// Let `kernel` use `bytes` of dynamic shared memory on the current device; asked once
// per device.
template <auto kernel>
cudaError_t allow_shared_memory(int bytes) {
  static std::atomic<unsigned long long> done{0};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

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

// ---- tensor-core path: bf16 / fp16, D = 128, D_keep 16 / 32 / 64, rows that TMA
// and 16-byte copies can take.  Three kernels: the prefix (shared_prefix.cu), the
// questions' text (shared_text.cu), and the join of their partial results
// (shared_merge.cu).  A partial result of a query row is (m, l, O[128]): the base-2
// maximum it is relative to, sum 2^(x - m) and sum 2^(x - m) v.

// How the prefix work is cut.  A unit is 128 query rows of one (prefix, KV head):
// rows (n, t, g) of its N questions, T tokens and G heads.  Its tokens come in
// blocks, 64 prompt tokens (weight 1) or 128 visual tokens (weight 2) each; the
// list of all units' blocks is cut into `grid` ranges of equal weight, one per CTA.
struct PrefixSplit {
  int rows;                  // N T G query rows of a (prefix, KV head)
  int row_tiles;             // ceil(rows / 128)
  int units;                 // P H_kv row_tiles
  int blocks_full, blocks_vis;
  int unit_start;            // weight of a unit's start and end (queries, rotation, partial result)
  int unit_weight;           // of a unit, its start included
  long long total;           // units * unit_weight
  int grid;

  __host__ __device__ int blocks() const { return blocks_full + blocks_vis; }
  // weight at which block j of a unit starts
  __host__ __device__ int block_start(int j) const {
    return unit_start + (j < blocks_full ? j : blocks_full + 2 * (j - blocks_full));
  }
  // first block of a unit that starts at weight >= w
  __host__ __device__ int block_from(int w) const {
    w -= unit_start;
    if (w <= 0) return 0;
    if (w <= blocks_full) return w;
    const int j = blocks_full + (w - blocks_full + 1) / 2;
    return j < blocks() ? j : blocks();
  }
  __host__ __device__ long long range_begin(int c) const { return (long long)c * total / grid; }
  // the CTA whose range holds weight w
  __host__ __device__ int owner(long long w) const { return (int)(((w + 1) * grid - 1) / total); }
  // CTAs that hold blocks of unit u.  Ranges are at least 2 long and block starts
  // at most 2 apart, so every CTA from the first to the last holds one.
  __host__ __device__ int first_cta(int u) const { return owner((long long)u * unit_weight + unit_start); }
  __host__ __device__ int last_cta(int u) const {
    return owner((long long)u * unit_weight + block_start(blocks() - 1));
  }
  // (unit, CTA) pairs lie on a staircase, so u + c numbers them without collision
  __host__ __device__ int slots() const { return units + grid; }
};

inline PrefixSplit prefix_split(long long prefixes, long long questions, long long tokens, long long groups,
                                long long kv_heads, long long seq_full, long long seq_sparse, long long text_cap, int sms) {
  PrefixSplit s;
  s.rows = (int)(questions * tokens * groups);
  s.row_tiles = (s.rows + 127) / 128;
  s.units = (int)(prefixes * kv_heads * s.row_tiles);
  s.blocks_full = (int)((seq_full + 63) / 64);
  s.blocks_vis = (int)((seq_sparse + 127) / 128);
  const long long weight = s.blocks_full + 2 * s.blocks_vis, all = s.units * weight;
  // Ranges of a few blocks: a quarter of the SMs is left to the text kernel, which then runs
  // beside this one instead of after it (8 questions on 16000 tokens: 20.6 us, 26.3 on all
  // SMs, 21.9 on half; ranges of many blocks cannot spare them: 123 us against 115, 700
  // against 600); half of them where the text is the larger part, 64 tokens of the caches
  // (half full) a weight (64 questions of 1024 tokens: 35.3, 37.8 with a quarter, 41.0 with none).
  const long long text = prefixes * questions * kv_heads * ((tokens * groups + 63) / 64) * text_cap / 64;
  if (text > 0 && all < 16ll * sms) sms -= text >= all ? sms / 2 : sms / 4;
  // A unit's start and end take 6 to 10 thousand cycles, where a block of 128 rows (weight 2)
  // takes 1800 and one of few rows two thirds of that: CTAs that meet a second unit get fewer blocks,
  // though not none.  (Weight 2 / this rule / 16: the whole attention in 21.2 / 20.6 / 20.6 us for
  // 56 rows of 4 heads with ranges of 9, 120.3 / 115.4 / 115.4 for 80 units of up to 128 rows,
  // 83.7 / 83.4 / 83.1 for 64 of 12; with one part of P 16 units with ranges of 2 13.5 / - / 14.5.)
  const long long range = all / sms;
  s.unit_start = (int)(range < 2 ? 2 : range > 16 ? 16 : range);
  s.unit_weight = (int)weight + s.unit_start;
  s.total = (long long)s.units * s.unit_weight;
  s.grid = (int)(s.total / 2 < sms ? (s.total / 2 > 0 ? s.total / 2 : 1) : sms);
  return s;
}

struct PrefixMaps {
  CUtensorMap kf, vf, ks, vs;   // 64-token boxes of the prompt, 128-token boxes of the visual span
};

struct PrefixParams {
  SharedParams s;
  PrefixSplit split;
  int R_layout;                 // R can be read 16 bytes at a time: 1 along its rows, 2 along its columns, 0 not
  float *ml, *acc;              // per slot: [128 rows][2] and [32 groups of 4 channels][128 rows][4]
  unsigned int *status;         // null: the device's own word
};
cudaError_t launch_shared_prefix(const PrefixMaps &maps, const PrefixParams &p, cudaStream_t stream);
// Address of the current device's status word, which calls that give none report to.
cudaError_t shared_status_address(void **address);

// Text: CTAs per (question, KV head, chunk of tokens, 16 or 64 query rows).  Chunks of 256
// tokens, so that few questions use many SMs; longer where that makes several waves of
// CTAs (the whole attention, 64 questions, 8 heads of 8 rows of 4096 tokens of 16 bits: 165 us
// with 256, 135 with 1024; 256 questions, 8 heads of 4 rows, 512 tokens: 82 and 76).  From 128 on:
// 8 questions of 640 tokens 20.6 us, of 2048 23.3, as from 256.
inline int text_chunk(long long batch, long long kv_heads, long long rows, long long cap) {
  const long long tiles = rows <= 16 ? 1 : (rows + 63) / 64;
  int chunk = 256;
  while (chunk < 1024 && batch * kv_heads * tiles * ((cap + chunk - 1) / chunk) > 148 * 8) chunk *= 2;
  return chunk;
}

struct TextParams {
  SharedParams s;
  int rows, chunk, chunks;      // T G query rows; tokens of a chunk, ceil(cap / chunk)
  int beside;                   // launched right after the prefix kernel, to run beside it
  float *ml, *acc;              // per (question, KV head, chunk): [rows][2] and [32 groups of 4 channels][rows][4]
};
cudaError_t launch_shared_text(const TextParams &p, cudaStream_t stream);

struct MergeParams {
  SharedParams s;
  PrefixSplit split;
  int has_prefix, has_text;
  int text_rows, text_chunk, text_chunks;
  const float *prefix_ml, *prefix_acc, *text_ml, *text_acc;
};
cudaError_t launch_shared_merge(const MergeParams &p, cudaStream_t stream);

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
// SMs of a device (capi.cu)
int device_sms(int device);

size_t verify_workspace_bytes(long long batch, long long drafts, long long vocab);
cudaError_t launch_verify(const VerifyParams &p, cudaStream_t stream);

}  // namespace rtk
