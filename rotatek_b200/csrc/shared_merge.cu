// Shared-prefix attention, the join: a query row's partial results -- one per CTA
// that held part of its prefix unit, one per text chunk of its question -- become
//   out = sum_i f_i O_i / sum_i f_i l_i,   f_i = 2^(m_i - max m),
// in slot order (the same result every time); a row that saw nothing is 0.
//
// Two kernels.  Where rows are many, a CTA takes 32 rows of a prefix unit: lane = row, so
// that a warp reads four channels of a partial of its unit, or of a question's text, in
// whole lines; it takes four such groups, so that the weights are worked out once for all
// four, and two partials in flight; the output goes out through shared memory.  Where
// rows are few and have many partials (few units on many SMs), a CTA takes a row.
#include "common.cuh"
#include "shared.h"

namespace rtk {
namespace {

// kQuads groups of four channels per thread, kDepth partials in flight.
template <typename T, int kQuads, int kDepth>
__global__ void __launch_bounds__(1024 / kQuads) shared_merge_kernel(const MergeParams p) {
  constexpr int kWarps = 32 / kQuads;
  __shared__ __align__(16) T out_s[32][128 + 8];
  const SharedParams &a = p.s;
  wait_for_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;    // channel groups warp + kWarps q
  const int u = blockIdx.x / 4, in_unit = (blockIdx.x % 4) * 32;
  const int ph = u / p.split.row_tiles, pre = ph / a.kv_heads, h = ph % a.kv_heads;
  const int base = (u % p.split.row_tiles) * 128 + in_unit;      // first row of the (prefix, KV head)
  if (base >= p.split.rows) return;
  const int r = base + lane;
  const bool live = r < p.split.rows;
  // row r is head g of token t of question n
  const int g = r % a.groups, nt = r / a.groups, t = nt % a.tokens, b = pre * a.questions + nt / a.tokens;

  float m = -INFINITY, l = 0.f;
  float4 o[kQuads];
#pragma unroll
  for (int q = 0; q < kQuads; ++q) o[q] = make_float4(0.f, 0.f, 0.f, 0.f);
  // `count` partials; ml(i), acc(i, q) their (m, l) and O of this row and a channel group
  auto join = [&](int count, auto ml, auto acc) {
    for (int first = 0; first < count; first += kDepth) {
      float2 e[kDepth];
      float4 v[kDepth][kQuads];
#pragma unroll
      for (int i = 0; i < kDepth; ++i) {
        const bool in = first + i < count;
        e[i] = in ? __ldcg(ml(first + i)) : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int q = 0; q < kQuads; ++q)
          v[i][q] = in ? __ldcg(acc(first + i, warp + kWarps * q)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float m2 = m;
#pragma unroll
      for (int i = 0; i < kDepth; ++i) m2 = fmaxf(m2, e[i].x);
      const float ref = m2 > -INFINITY ? m2 : 0.f;
      const float f = fast_exp2(m - ref);            // nothing yet: 0
      m = m2;
      l *= f;
#pragma unroll
      for (int q = 0; q < kQuads; ++q) {
        o[q].x *= f;
        o[q].y *= f;
        o[q].z *= f;
        o[q].w *= f;
      }
#pragma unroll
      for (int i = 0; i < kDepth; ++i) {
        const float w = fast_exp2(e[i].x - ref);
        if (w == 0.f) continue;                      // a partial that saw nothing: its O may be anything
        l = fmaf(w, e[i].y, l);
#pragma unroll
        for (int q = 0; q < kQuads; ++q) {
          o[q].x = fmaf(w, v[i][q].x, o[q].x);
          o[q].y = fmaf(w, v[i][q].y, o[q].y);
          o[q].z = fmaf(w, v[i][q].z, o[q].z);
          o[q].w = fmaf(w, v[i][q].w, o[q].w);
        }
      }
    }
  };
  if (live && p.has_prefix) {
    const int c0 = p.split.first_cta(u);
    const long long slot = u + c0;
    const float2 *ml = reinterpret_cast<const float2 *>(p.prefix_ml) + slot * 128 + in_unit + lane;
    const float4 *acc = reinterpret_cast<const float4 *>(p.prefix_acc) + slot * 4096 + in_unit + lane;
    join(p.split.last_cta(u) - c0 + 1, [&](int i) { return ml + i * 128; },
         [&](int i, int c4) { return acc + (i * 32ll + c4) * 128; });
  }
  if (live && p.has_text) {
    const int len = min(max(a.lens[b * a.lens_s], 0), a.cap), row = t * a.groups + g;
    const long long first = ((long long)b * a.kv_heads + h) * p.text_chunks;
    const float2 *ml = reinterpret_cast<const float2 *>(p.text_ml) + first * p.text_rows + row;
    const float4 *acc = reinterpret_cast<const float4 *>(p.text_acc) + first * 32 * p.text_rows + row;
    join((len + p.text_chunk - 1) / p.text_chunk, [&](int i) { return ml + (long long)i * p.text_rows; },
         [&](int i, int c4) { return acc + (i * 32ll + c4) * p.text_rows; });
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int q = 0; q < kQuads; ++q)
    *reinterpret_cast<uint2 *>(&out_s[lane][(warp + kWarps * q) * 4]) =
        make_uint2(pack2<T>(o[q].x * inv, o[q].y * inv), pack2<T>(o[q].z * inv, o[q].w * inv));
  __syncthreads();
  // warp = row, lane = four channels
  for (int i = warp; i < 32; i += kWarps) {
    const int r2 = base + i;
    if (r2 >= p.split.rows) return;
    const int g2 = r2 % a.groups, nt2 = r2 / a.groups, t2 = nt2 % a.tokens, b2 = pre * a.questions + nt2 / a.tokens;
    T *out = static_cast<T *>(a.out) + b2 * a.o_s[0] + t2 * a.o_s[1] + (h * a.groups + g2) * a.o_s[2] + lane * 4 * a.o_s[3];
    const T *from = &out_s[i][lane * 4];
    if (a.o_s[3] == 1 && reinterpret_cast<uintptr_t>(out) % 8 == 0) {
      *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<const uint2 *>(from);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) out[k * a.o_s[3]] = from[k];
    }
  }
}

// Few units on many SMs: a CTA per row, lane = four channels.  Its four warps take a quarter
// of the partials each -- their (m, l) 32 at a time, a lane each, their O with eight
// loads in flight -- and are joined in warp order.
template <typename T>
__global__ void __launch_bounds__(128) shared_merge_rows_kernel(const MergeParams p) {
  const SharedParams &a = p.s;
  wait_for_previous();
  __shared__ float2 ml_s[4];
  __shared__ float4 o_s[4][32];
  const long long idx = blockIdx.x;
  const int lane = threadIdx.x & 31;
  const int hq = (int)(idx % a.q_heads);
  const long long bt = idx / a.q_heads;
  const int t = (int)(bt % a.tokens), b = (int)(bt / a.tokens);
  const int h = hq / a.groups, g = hq % a.groups;

  // partial i: the prefix's CTAs first, then the text's chunks
  int prefixes = 0, total = 0;
  long long at_p = 0, at_t = 0, slot0 = 0, text0 = 0, r0 = 0;
  if (p.has_prefix) {
    const int pre = b / a.questions, n = b % a.questions;
    const int r = (n * a.tokens + t) * a.groups + g;
    const int u = (pre * a.kv_heads + h) * p.split.row_tiles + r / 128;
    const int c0 = p.split.first_cta(u);
    prefixes = p.split.last_cta(u) - c0 + 1;
    slot0 = u + c0;
    r0 = r % 128;
    at_p = slot0 * 128 + r0;
  }
  total = prefixes;
  if (p.has_text) {
    const int len = min(max(a.lens[b * a.lens_s], 0), a.cap);
    total += (len + p.text_chunk - 1) / p.text_chunk;
    text0 = ((long long)b * a.kv_heads + h) * p.text_chunks;
    at_t = text0 * p.text_rows + t * a.groups + g;
  }
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  const int warp = threadIdx.x >> 5, quarter = (total + 3) / 4, last = min(total, (warp + 1) * quarter);
  for (int first = warp * quarter; first < last; first += 32) {
    const int count = min(32, last - first);
    float2 ml = make_float2(-INFINITY, 0.f);
    const float *src = nullptr;
    int stride = 0;                                   // from one group of four channels to the next
    if (lane < count) {
      const int i = first + lane;
      if (i < prefixes) {
        ml = __ldcg(reinterpret_cast<const float2 *>(p.prefix_ml) + at_p + i * 128ll);
        src = p.prefix_acc + ((slot0 + i) * 32 * 128 + r0) * 4;
        stride = 128 * 4;
      } else {
        const long long at = at_t + (long long)(i - prefixes) * p.text_rows;
        ml = __ldcg(reinterpret_cast<const float2 *>(p.text_ml) + at);
        src = p.text_acc + ((text0 + i - prefixes) * 32 * p.text_rows + t * a.groups + g) * 4;
        stride = p.text_rows * 4;
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
        const int st = __shfl_sync(0xffffffffu, stride, from);
        if (i + k >= count) wi[k] = 0.f;
        v[k] = wi[k] != 0.f ? __ldcg(reinterpret_cast<const float4 *>(q + (long long)lane * st)) : make_float4(0.f, 0.f, 0.f, 0.f);
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
  if (lane == 0) ml_s[warp] = make_float2(m, l);
  o_s[warp][lane] = o;
  __syncthreads();
  if (warp > 0) return;
  float top = m;
#pragma unroll
  for (int w = 1; w < 4; ++w) top = fmaxf(top, ml_s[w].x);
  l = 0.f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (!(ml_s[w].x > -INFINITY)) continue;
    const float f = fast_exp2(ml_s[w].x - top);
    const float4 v = o_s[w][lane];
    l = fmaf(f, ml_s[w].y, l);
    o.x = fmaf(f, v.x, o.x);
    o.y = fmaf(f, v.y, o.y);
    o.z = fmaf(f, v.z, o.z);
    o.w = fmaf(f, v.w, o.w);
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

template <typename T>
cudaError_t launch(const MergeParams &p, cudaStream_t stream) {
  const dim3 grid((unsigned)p.split.units * 4u);
  // partials of a row from the prefix: about grid / units
  if (p.split.grid > 4 * p.split.units) {
    const long long rows = (long long)p.s.prefixes * p.s.questions * p.s.tokens * p.s.q_heads;
    return launch_overlapping(shared_merge_rows_kernel<T>, dim3((unsigned)rows), dim3(128), 0, stream, p);
  }
  return launch_overlapping(shared_merge_kernel<T, 4, 2>, grid, dim3(256), 0, stream, p);
}

}  // namespace

cudaError_t launch_shared_merge(const MergeParams &p, cudaStream_t stream) {
  return p.s.dtype == 1 ? launch<__nv_bfloat16>(p, stream) : launch<__half>(p, stream);
}

}  // namespace rtk
