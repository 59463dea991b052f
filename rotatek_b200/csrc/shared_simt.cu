// Generic kernel of the shared-prefix attention (CUDA cores, fp32 arithmetic):
// fp32 tensors, any head width up to 256, any D_keep, any strides.
//
// For query row (b, t, h) of prefix p = b / questions, in base 2 with
// c = log2(e) / sqrt(D):
//   visual token    x = c (sum_j (q R)_j k~_j + q . delta_mu)
//   prompt token    x = c q . k            where mask != 0
//   text token s    x = c q . k_text       where s < len[b] - (T - 1 - t)
//   out = sum 2^(x - m) v / sum 2^(x - m),  m = max x;  0 where nothing is seen
//
// One CTA per row; its four warps take every fourth token, one logit per step
// by a shuffle sum over the channels, and keep a running (m, l, acc) each in
// fp32; the warps' states are merged in shared memory in warp order.  Tokens
// that a row does not see are never read, so what lies there (infinities, NaN,
// memory never written) cannot reach an output.  Nothing here is tuned: it is
// the kernel that is right for every layout.
#include "common.cuh"
#include "shared.h"

#include <cuda_fp8.h>

namespace rtk {
namespace {

constexpr int kWarps = 4;
constexpr int kMaxD = 256;

template <typename T>
__device__ __forceinline__ float ld(const void *base, long long off) {
  return to_f32(reinterpret_cast<const T *>(base)[off]);
}

__device__ __forceinline__ float ld_e4m3(const void *base, long long off) {
  __nv_fp8_e4m3 v;
  v.__x = reinterpret_cast<const unsigned char *>(base)[off];
  return static_cast<float>(v);
}

struct RowState {
  float m, l;
  float acc[kMaxD / 32];
};

// one token: its logit is complete in every lane; v(d) gives channel d of its Value
template <typename F>
__device__ __forceinline__ void step(RowState &st, float x, int D, int lane, F v) {
  if (!(x > -INFINITY) && !isnan(x)) return;        // weight 0
  float keep = 1.f;
  if (x > st.m) {
    keep = exp2f(st.m - x);                          // first token: 2^-inf = 0
    st.m = x;
  }
  const float w = exp2f(x - st.m);
  st.l = fmaf(st.l, keep, w);
#pragma unroll
  for (int i = 0; i < kMaxD / 32; ++i) {
    const int d = lane + 32 * i;
    if (d < D) st.acc[i] = fmaf(st.acc[i], keep, w * v(d));
  }
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) shared_simt_kernel(const SharedParams p) {
  __shared__ float q_s[kMaxD], qrot_s[kMaxD], red_s[kWarps];
  __shared__ float m_s[kWarps], l_s[kWarps], acc_s[kWarps][kMaxD];

  const int h = blockIdx.x % p.q_heads;
  const int bt = blockIdx.x / p.q_heads;
  const int t = bt % p.tokens, b = bt / p.tokens;
  const int pre = b / p.questions, kvh = h / p.groups;
  const int D = p.head_dim, DK = p.head_dim_keep;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  for (int d = threadIdx.x; d < D; d += blockDim.x)
    q_s[d] = ld<T>(p.q.data, b * p.q.s[0] + t * p.q.s[1] + h * p.q.s[2] + d * p.q.s[3]);
  __syncthreads();
  if (p.seq_sparse > 0) {
    const long long rb = pre * p.R.s[0] + kvh * p.R.s[1];
    for (int j = threadIdx.x; j < DK; j += blockDim.x) {
      float a = 0.f;
      for (int d = 0; d < D; ++d) a = fmaf(q_s[d], ld<T>(p.R.data, rb + d * p.R.s[2] + j * p.R.s[3]), a);
      qrot_s[j] = a;
    }
  }
  float bias = 0.f;
  if (p.dm.data != nullptr && p.seq_sparse > 0) {
    const long long db = pre * p.dm.s[0] + kvh * p.dm.s[1];
    for (int d = threadIdx.x; d < D; d += blockDim.x) bias = fmaf(q_s[d], ld<T>(p.dm.data, db + d * p.dm.s[2]), bias);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) bias += __shfl_xor_sync(0xffffffffu, bias, o);
  if (lane == 0) red_s[warp] = bias;
  __syncthreads();
  bias = 0.f;
  for (int w = 0; w < kWarps; ++w) bias += red_s[w];

  RowState st;
  st.m = -INFINITY;
  st.l = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxD / 32; ++i) st.acc[i] = 0.f;
  const float c = p.scale_log2;

  // prompt
  for (int s = warp; s < p.seq_full; s += kWarps) {
    if (p.mask.data != nullptr &&
        static_cast<const uint8_t *>(p.mask.data)[pre * p.mask.s[0] + s * p.mask.s[1]] == 0)
      continue;
    const long long kb = pre * p.kf.s[0] + kvh * p.kf.s[1] + s * p.kf.s[2];
    float x = 0.f;
    for (int d = lane; d < D; d += 32) x = fmaf(q_s[d], ld<T>(p.kf.data, kb + d * p.kf.s[3]), x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    const long long vb = pre * p.vf.s[0] + kvh * p.vf.s[1] + s * p.vf.s[2];
    step(st, x * c, D, lane, [&](int d) { return ld<T>(p.vf.data, vb + d * p.vf.s[3]); });
  }
  // visual span
  for (int s = warp; s < p.seq_sparse; s += kWarps) {
    const long long kb = pre * p.ks.s[0] + kvh * p.ks.s[1] + s * p.ks.s[2];
    float x = 0.f;
    for (int j = lane; j < DK; j += 32) x = fmaf(qrot_s[j], ld<T>(p.ks.data, kb + j * p.ks.s[3]), x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    const long long vb = pre * p.vs.s[0] + kvh * p.vs.s[1] + s * p.vs.s[2];
    step(st, (x + bias) * c, D, lane, [&](int d) { return ld<T>(p.vs.data, vb + d * p.vs.s[3]); });
  }
  // the question's own text, up to the tokens query t sees
  const int len = p.cap > 0 ? min(max(p.lens[b * p.lens_s], 0), p.cap) : 0;
  const int seen = len - (p.tokens - 1 - t);
  for (int s = warp; s < seen; s += kWarps) {
    const long long kb = b * p.kt.s[0] + kvh * p.kt.s[1] + s * p.kt.s[2];
    const long long vb = b * p.vt.s[0] + kvh * p.vt.s[1] + s * p.vt.s[2];
    float x = 0.f;
    if (p.text_fp8) {
      for (int d = lane; d < D; d += 32) x = fmaf(q_s[d], ld_e4m3(p.kt.data, kb + d * p.kt.s[3]), x);
    } else {
      for (int d = lane; d < D; d += 32) x = fmaf(q_s[d], ld<T>(p.kt.data, kb + d * p.kt.s[3]), x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (p.text_fp8) {
      const float kscale = static_cast<const float *>(p.ksc.data)[b * p.ksc.s[0] + kvh * p.ksc.s[1] + s * p.ksc.s[2]];
      const float vscale = static_cast<const float *>(p.vsc.data)[b * p.vsc.s[0] + kvh * p.vsc.s[1] + s * p.vsc.s[2]];
      step(st, x * kscale * c, D, lane, [&](int d) { return vscale * ld_e4m3(p.vt.data, vb + d * p.vt.s[3]); });
    } else {
      step(st, x * c, D, lane, [&](int d) { return ld<T>(p.vt.data, vb + d * p.vt.s[3]); });
    }
  }

  if (lane == 0) {
    m_s[warp] = st.m;
    l_s[warp] = st.l;
  }
#pragma unroll
  for (int i = 0; i < kMaxD / 32; ++i)
    if (lane + 32 * i < D) acc_s[warp][lane + 32 * i] = st.acc[i];
  __syncthreads();
  float m = -INFINITY, l = 0.f;
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, m_s[w]);
  float f[kWarps];
  for (int w = 0; w < kWarps; ++w) {
    f[w] = m_s[w] > -INFINITY ? exp2f(m_s[w] - m) : 0.f;
    l = fmaf(l_s[w], f[w], l);
  }
  T *out = static_cast<T *>(p.out) + b * p.o_s[0] + t * p.o_s[1] + h * p.o_s[2];
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float a = 0.f;
    for (int w = 0; w < kWarps; ++w) a = fmaf(acc_s[w][d], f[w], a);
    out[d * p.o_s[3]] = from_f32<T>(l != 0.f ? a / l : 0.f);
  }
}

}  // namespace

cudaError_t launch_shared_simt(const SharedParams &p, cudaStream_t stream) {
  const long long rows = (long long)p.prefixes * p.questions * p.tokens * p.q_heads;
  if (rows == 0) return cudaSuccess;
  const dim3 grid((unsigned)rows), block(kWarps * 32);
  if (p.dtype == 0) shared_simt_kernel<float><<<grid, block, 0, stream>>>(p);
  else if (p.dtype == 1) shared_simt_kernel<__nv_bfloat16><<<grid, block, 0, stream>>>(p);
  else shared_simt_kernel<__half><<<grid, block, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace rtk
