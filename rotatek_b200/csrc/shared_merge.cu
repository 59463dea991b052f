// Shared-prefix attention, the join: a query row's partial results -- one per CTA
// that held part of its prefix unit, one per text chunk of its question -- become
//   out = sum_i f_i O_i / sum_i f_i l_i,   f_i = 2^(m_i - max m),
// in slot order (the same result every time); a row that saw nothing is 0.
//
// One warp per row, lane = 4 channels.  A row can have as many partials as there are
// SMs, so their (m, l) are read 32 at a time, a lane each, and their O with eight loads
// in flight; partials come from L2 mostly.
#include "common.cuh"
#include "shared.h"

namespace rtk {
namespace {

constexpr int kWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) shared_merge_kernel(const MergeParams p) {
  const SharedParams &a = p.s;
  wait_for_previous();
  const long long rows = (long long)a.prefixes * a.questions * a.tokens * a.q_heads;
  const long long idx = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (idx >= rows) return;
  const int lane = threadIdx.x & 31;
  const int hq = (int)(idx % a.q_heads);
  const long long bt = idx / a.q_heads;
  const int t = (int)(bt % a.tokens), b = (int)(bt / a.tokens);
  const int h = hq / a.groups, g = hq % a.groups;

  // partial i: the prefix's CTAs first, then the text's chunks
  int prefixes = 0, total = 0;
  long long at_p = 0, at_t = 0;
  if (p.has_prefix) {
    const int pre = b / a.questions, n = b % a.questions;
    const int r = (n * a.tokens + t) * a.groups + g;
    const int u = (pre * a.kv_heads + h) * p.split.row_tiles + r / 128;
    const int c0 = p.split.first_cta(u);
    prefixes = p.split.last_cta(u) - c0 + 1;
    at_p = (long long)(u + c0) * 128 + r % 128;
  }
  total = prefixes;
  if (p.has_text) {
    const int len = min(max(a.lens[b * a.lens_s], 0), a.cap);
    total += (len + kTextChunk - 1) / kTextChunk;
    at_t = ((long long)b * a.kv_heads + h) * p.text_chunks * p.text_rows + t * a.groups + g;
  }
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int first = 0; first < total; first += 32) {
    const int count = min(32, total - first);
    float2 ml = make_float2(-INFINITY, 0.f);
    const float *src = nullptr;
    if (lane < count) {
      const int i = first + lane;
      if (i < prefixes) {
        ml = __ldcg(reinterpret_cast<const float2 *>(p.prefix_ml) + at_p + i * 128ll);
        src = p.prefix_acc + (at_p + i * 128ll) * 128;
      } else {
        const long long at = at_t + (long long)(i - prefixes) * p.text_rows;
        ml = __ldcg(reinterpret_cast<const float2 *>(p.text_ml) + at);
        src = p.text_acc + at * 128;
      }
    }
    float top = ml.x;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    const float m2 = fmaxf(m, top), base = m2 > -INFINITY ? m2 : 0.f;
    const float f = fast_exp2(m - base);              // nothing yet: 0
    float w = fast_exp2(ml.x - base);                 // an empty partial: 0
    float sum = w > 0.f || isnan(w) ? w * ml.y : 0.f;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    m = m2;
    l = fmaf(l, f, sum);
    o.x *= f;
    o.y *= f;
    o.z *= f;
    o.w *= f;
    for (int i = 0; i < count; i += 8) {
      float4 v[8];
      float wi[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int from = i + k < count ? i + k : i;
        wi[k] = __shfl_sync(0xffffffffu, w, from);
        const float *q = reinterpret_cast<const float *>(__shfl_sync(0xffffffffu, reinterpret_cast<long long>(src), from));
        if (i + k >= count) wi[k] = 0.f;
        v[k] = wi[k] != 0.f ? __ldcg(reinterpret_cast<const float4 *>(q + lane * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {                   // an empty partial's O was never written
        o.x = fmaf(wi[k], v[k].x, o.x);
        o.y = fmaf(wi[k], v[k].y, o.y);
        o.z = fmaf(wi[k], v[k].z, o.z);
        o.w = fmaf(wi[k], v[k].w, o.w);
      }
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  T *out = static_cast<T *>(a.out) + b * a.o_s[0] + t * a.o_s[1] + hq * a.o_s[2] + lane * 4 * a.o_s[3];
  const float v[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  if (a.o_s[3] == 1 && reinterpret_cast<uintptr_t>(out) % 8 == 0) {
    *reinterpret_cast<uint2 *>(out) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i * a.o_s[3]] = from_f32<T>(v[i]);
  }
}

}  // namespace

cudaError_t launch_shared_merge(const MergeParams &p, cudaStream_t stream) {
  const long long rows = (long long)p.s.prefixes * p.s.questions * p.s.tokens * p.s.q_heads;
  const unsigned grid = (unsigned)((rows + kWarps - 1) / kWarps);
  return p.s.dtype == 1 ? launch_overlapping(shared_merge_kernel<__nv_bfloat16>, dim3(grid), dim3(kWarps * 32), 0, stream, p)
                        : launch_overlapping(shared_merge_kernel<__half>, dim3(grid), dim3(kWarps * 32), 0, stream, p);
}

}  // namespace rtk
