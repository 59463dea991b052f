// Shared-prefix attention, the join: a query row's partial results -- one per CTA
// that held part of its prefix unit, one per text chunk of its question -- become
//   out = sum_i f_i O_i / sum_i f_i l_i,   f_i = 2^(m_i - max m),
// in slot order (the same result every time); a row that saw nothing is 0.
//
// One warp per row, lane = 4 channels.  The partials are read once, from L2 mostly.
#include "common.cuh"
#include "shared.h"

namespace rtk {
namespace {

constexpr int kWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) shared_merge_kernel(const MergeParams p) {
  const SharedParams &a = p.s;
  const long long rows = (long long)a.prefixes * a.questions * a.tokens * a.q_heads;
  const long long idx = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (idx >= rows) return;
  const int lane = threadIdx.x & 31;
  const int hq = (int)(idx % a.q_heads);
  const long long bt = idx / a.q_heads;
  const int t = (int)(bt % a.tokens), b = (int)(bt / a.tokens);
  const int h = hq / a.groups, g = hq % a.groups;

  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto take = [&](float2 ml, const float *src) {
    if (!(ml.x > -INFINITY) && !isnan(ml.x)) return;
    const float m2 = fmaxf(m, ml.x);
    const float f = fast_exp2(m - m2), fi = fast_exp2(ml.x - m2);
    m = m2;
    l = fmaf(l, f, ml.y * fi);
    const float4 v = *reinterpret_cast<const float4 *>(src + lane * 4);
    o.x = fmaf(o.x, f, v.x * fi);
    o.y = fmaf(o.y, f, v.y * fi);
    o.z = fmaf(o.z, f, v.z * fi);
    o.w = fmaf(o.w, f, v.w * fi);
  };
  if (p.has_prefix) {
    const int pre = b / a.questions, n = b % a.questions;
    const int r = (n * a.tokens + t) * a.groups + g;
    const int u = (pre * a.kv_heads + h) * p.split.row_tiles + r / 128;
    const int c1 = p.split.last_cta(u);
    for (int c = p.split.first_cta(u); c <= c1; ++c) {
      const long long at = (long long)(u + c) * 128 + r % 128;
      take(reinterpret_cast<const float2 *>(p.prefix_ml)[at], p.prefix_acc + at * 128);
    }
  }
  if (p.has_text) {
    const int len = min(max(a.lens[b * a.lens_s], 0), a.cap);
    const int r = t * a.groups + g;
    for (int c = 0; c * kTextChunk < len; ++c) {
      const long long at = (((long long)b * a.kv_heads + h) * p.text_chunks + c) * p.text_rows + r;
      take(reinterpret_cast<const float2 *>(p.text_ml)[at], p.text_acc + at * 128);
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
  if (p.s.dtype == 1) shared_merge_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, stream>>>(p);
  else shared_merge_kernel<__half><<<grid, kWarps * 32, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace rtk
