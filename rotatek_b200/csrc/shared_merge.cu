// Shared-prefix attention, the join: a query row's partial results -- one per CTA
// that held part of its prefix unit, one per text chunk of its question -- become
//   out = sum_i f_i O_i / sum_i f_i l_i,   f_i = 2^(m_i - max m),
// in slot order (the same result every time); a row that saw nothing is 0.
//
// Two kernels, both launched while the partials are still being made: what does not depend on
// them (where a row's partials lie) is worked out before the wait.  Where rows are many, a CTA
// takes 32 rows of a prefix unit: lane = row, so that a warp reads four channels of a partial
// of its unit, or of a question's text, in whole lines; it takes four such groups, so that the
// weights are worked out once for all four, and two partials in flight; the output goes out
// through shared memory.  Where that would leave SMs idle, CTAs of 8 rows and 32 channels
// whose warps split the partials.
//
// Measured, the whole attention with tiles of 32 rows / of 8: 1024 working CTAs of 32 rows 600 /
// 683 us, 288 of them 115 / 139, 128: 102.9 / 102.5, 64: 83.0 / 82.8 and 61.1 / 60.7, 16: 34.5 /
// 27.5, 8: 28.7 / 20.6.
//
// What bounds it: after the last partial, latency (2 to 4 us); with the many rows of the first
// case its bytes, 61 MB of partials and 8 of output, mostly from L2.
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
        if (e[i].x == -INFINITY) continue;           // a partial that saw nothing: its O may be anything
        const float w = fast_exp2(e[i].x - ref);     // 0 times NaN stays NaN
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
  int prefixes = 0, chunks = 0;
  long long slot = 0, first = 0;
  const int row = t * a.groups + g;
  if (live && p.has_prefix) {
    const int c0 = p.split.first_cta(u);
    prefixes = p.split.last_cta(u) - c0 + 1;
    slot = u + c0;
  }
  if (live && p.has_text) {
    const int len = min(max(a.lens[b * a.lens_s], 0), a.cap);
    chunks = (len + p.text_chunk - 1) / p.text_chunk;
    first = ((long long)b * a.kv_heads + h) * p.text_chunks;
  }
  wait_for_previous();                               // where the partials are is known by then
  const float2 *ml_p = reinterpret_cast<const float2 *>(p.prefix_ml) + slot * 128 + in_unit + lane;
  const float4 *acc_p = reinterpret_cast<const float4 *>(p.prefix_acc) + slot * 4096 + in_unit + lane;
  join(prefixes, [&](int i) { return ml_p + i * 128; }, [&](int i, int c4) { return acc_p + (i * 32ll + c4) * 128; });
  const float2 *ml_t = reinterpret_cast<const float2 *>(p.text_ml) + first * p.text_rows + row;
  const float4 *acc_t = reinterpret_cast<const float4 *>(p.text_acc) + first * 32 * p.text_rows + row;
  join(chunks, [&](int i) { return ml_t + (long long)i * p.text_rows; },
       [&](int i, int c4) { return acc_t + (i * 32ll + c4) * p.text_rows; });
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

// Few units on many SMs: a row has many partials.  A CTA takes 8 rows of a unit and 8 groups
// of four channels; a warp's load is 4 groups of 8 rows (whole lines: a CTA per row, with
// lane = group, asked for 32 lines per load, and where CTAs crowded on the SMs that the prefix
// had left free they queued for 5 us).  Two warps side by side, four pairs for every fourth
// partial each, eight partials in flight; the pairs are joined in order.
constexpr int kSplitRows = 8, kSplitWays = 4, kSplitDepth = 8;

template <typename T>
__global__ void __launch_bounds__(64 * kSplitWays) shared_merge_split_kernel(const MergeParams p) {
  __shared__ float2 ml_s[kSplitWays][kSplitRows];
  __shared__ float4 o_s[kSplitWays][64];
  const SharedParams &a = p.s;
  const int lane = threadIdx.x & 31, side = (threadIdx.x >> 5) & 1, way = threadIdx.x >> 6;
  const int groups = (min(p.split.rows, 128) + kSplitRows - 1) / kSplitRows;      // of rows, in a unit
  const int c4 = (blockIdx.x & 3) * 8 + side * 4 + (lane >> 3);                   // group of four channels
  const int u = (int)(blockIdx.x >> 2) / groups, in_unit = (int)(blockIdx.x >> 2) % groups * kSplitRows;
  const int ph = u / p.split.row_tiles, pre = ph / a.kv_heads, h = ph % a.kv_heads;
  const int r = (u % p.split.row_tiles) * 128 + in_unit + (lane & 7);
  const bool live = r < p.split.rows;
  // row r is head g of token t of question n
  const int g = r % a.groups, nt = r / a.groups, t = nt % a.tokens, b = pre * a.questions + nt / a.tokens;

  // partial i: the prefix's CTAs first, then the text's chunks
  int prefixes = 0, total = 0;
  const float2 *ml_p = nullptr, *ml_t = nullptr;
  const float4 *acc_p = nullptr, *acc_t = nullptr;
  if (live && p.has_prefix) {
    const int c0 = p.split.first_cta(u);
    prefixes = p.split.last_cta(u) - c0 + 1;
    const long long slot = u + c0;
    ml_p = reinterpret_cast<const float2 *>(p.prefix_ml) + slot * 128 + r % 128;
    acc_p = reinterpret_cast<const float4 *>(p.prefix_acc) + (slot * 32 + c4) * 128 + r % 128;
  }
  total = prefixes;
  if (live && p.has_text) {
    const int len = min(max(a.lens[b * a.lens_s], 0), a.cap), row = t * a.groups + g;
    total += (len + p.text_chunk - 1) / p.text_chunk;
    const long long first = ((long long)b * a.kv_heads + h) * p.text_chunks;
    ml_t = reinterpret_cast<const float2 *>(p.text_ml) + first * p.text_rows + row;
    acc_t = reinterpret_cast<const float4 *>(p.text_acc) + (first * 32 + c4) * p.text_rows + row;
  }
  wait_for_previous();

  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int first = way; first < total; first += kSplitWays * kSplitDepth) {
    float2 e[kSplitDepth];
    float4 v[kSplitDepth];
#pragma unroll
    for (int k = 0; k < kSplitDepth; ++k) {
      const int i = first + kSplitWays * k;
      e[k] = make_float2(-INFINITY, 0.f);
      if (i < prefixes) {
        e[k] = __ldcg(ml_p + i * 128);
        v[k] = __ldcg(acc_p + i * 4096ll);
      } else if (i < total) {
        e[k] = __ldcg(ml_t + (long long)(i - prefixes) * p.text_rows);
        v[k] = __ldcg(acc_t + (i - prefixes) * 32ll * p.text_rows);
      }
    }
    float m2 = m;
#pragma unroll
    for (int k = 0; k < kSplitDepth; ++k) m2 = fmaxf(m2, e[k].x);
    const float ref = m2 > -INFINITY ? m2 : 0.f;
    const float f = fast_exp2(m - ref);              // nothing yet: 0
    m = m2;
    l *= f;
    o.x *= f;
    o.y *= f;
    o.z *= f;
    o.w *= f;
#pragma unroll
    for (int k = 0; k < kSplitDepth; ++k) {
      if (e[k].x == -INFINITY) continue;             // a partial that saw nothing: its O may be anything
      const float w = fast_exp2(e[k].x - ref);       // 0 times NaN stays NaN
      l = fmaf(w, e[k].y, l);
      o.x = fmaf(w, v[k].x, o.x);
      o.y = fmaf(w, v[k].y, o.y);
      o.z = fmaf(w, v[k].z, o.z);
      o.w = fmaf(w, v[k].w, o.w);
    }
  }
  if (side == 0 && lane < kSplitRows) ml_s[way][lane] = make_float2(isnan(l) ? l : m, l);
  o_s[way][side * 32 + lane] = o;
  __syncthreads();
  if (way > 0 || !live) return;
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kSplitWays; ++w) top = fmaxf(top, ml_s[w][lane & 7].x);
  const float ref = top > -INFINITY ? top : 0.f;
  l = 0.f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < kSplitWays; ++w) {
    const float2 e = ml_s[w][lane & 7];
    const float f = fast_exp2(e.x - ref);            // nothing there: 0
    const float4 v = o_s[w][side * 32 + lane];
    l = fmaf(f, e.y, l);
    o.x = fmaf(f, v.x, o.x);
    o.y = fmaf(f, v.y, o.y);
    o.z = fmaf(f, v.z, o.z);
    o.w = fmaf(f, v.w, o.w);
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  T *out = static_cast<T *>(a.out) + b * a.o_s[0] + t * a.o_s[1] + (h * a.groups + g) * a.o_s[2] + c4 * 4 * a.o_s[3];
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
  const int rows = p.split.rows < 128 ? p.split.rows : 128;        // of a unit
  if (p.split.units * ((rows + 31) / 32) < 96)                     // 32-row CTAs with work
    return launch_overlapping(shared_merge_split_kernel<T>,
                              dim3((unsigned)p.split.units * ((rows + kSplitRows - 1) / kSplitRows) * 4),
                              dim3(64 * kSplitWays), 0, stream, p);
  const dim3 grid((unsigned)p.split.units * 4u);
  return launch_overlapping(shared_merge_kernel<T, 4, 2>, grid, dim3(256), 0, stream, p);
}

}  // namespace

cudaError_t launch_shared_merge(const MergeParams &p, cudaStream_t stream) {
  return p.s.dtype == 1 ? launch<__nv_bfloat16>(p, stream) : launch<__half>(p, stream);
}

}  // namespace rtk
