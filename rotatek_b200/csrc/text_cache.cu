// Text caches of the questions that share a prefix: new Keys and Values written
// at each question's own length (as e4m3 with a scale per row, or as they are),
// and 8-bit caches read back.
//
//   amax  = largest finite |x| of the row (b, h, token) over its D channels
//   scale = max(amax / 448, 2^-126), 1 for a row without one
//   x8    = e4m3(x / scale): fp32 division rounded to nearest, then to the
//           nearest e4m3 value (ties to even); +-infinity is stored as +-448, NaN
//           as NaN
//   read  = round(x8 * scale) once to the output's type; 0 past the length
//
// A scale for each row, not for a channel of the whole span: a row is final when
// it is written, so appending never touches what is already there.
//
// Both are bound by HBM.  Rows of 128 channels with 16-byte aligned, unit-stride
// channels take 16-byte accesses and keep several rows of each thread in flight;
// anything else takes the scalar kernels below them.
#include "common.cuh"
#include "shared.h"

#include <cuda_fp8.h>

namespace rtk {
namespace {

constexpr float kE4m3Max = 448.f;

__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;     // NaN compares false
}

__device__ __forceinline__ float row_scale(float amax) {
  return amax > 0.f ? fmaxf(__fdiv_rn(amax, kE4m3Max), 1.17549435e-38f) : 1.f;
}

// Row r of the append: which cache (0 Keys, 1 Values), question, token, head.
// Heads run fastest, the order in which a fused projection leaves the rows.
struct AppendRow {
  int side, b, t, h, pos;
  bool live;
};

__device__ __forceinline__ AppendRow append_row(const AppendParams &p, unsigned r, unsigned total) {
  AppendRow a;
  a.live = r < 2u * total;
  if (!a.live) r = 0;
  a.side = r >= total;
  unsigned i = a.side ? r - total : r;
  a.h = i % p.heads;
  i /= p.heads;
  a.t = i % p.tokens;
  a.b = i / p.tokens;
  a.pos = p.lens[a.b * p.lens_s] + a.t;
  const int count = p.counts != nullptr ? p.counts[a.b * p.counts_s] : p.tokens;
  a.live = a.live && a.t < count && a.pos >= 0 && a.pos < p.cap;
  return a;
}

__device__ __forceinline__ long long row_offset(const SharedTensor &x, int b, int h, int s) {
  return b * x.s[0] + h * x.s[1] + s * x.s[2];
}

// 8 channels of a row as floats (16 or 32 bytes)
template <typename T>
struct Eight {
  uint4 raw[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *src) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = __ldg(reinterpret_cast<const uint4 *>(src) + i);
  }
  __device__ __forceinline__ void store(T *dst) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4 *>(dst)[i] = raw[i];
  }
  __device__ __forceinline__ void floats(float (&f)[8]) const {
    if constexpr (sizeof(T) == 4) {
      const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
    } else {
      unpack2<T>(raw[0].x, f[0], f[1]);
      unpack2<T>(raw[0].y, f[2], f[3]);
      unpack2<T>(raw[0].z, f[4], f[5]);
      unpack2<T>(raw[0].w, f[6], f[7]);
    }
  }
};

// D = 128: 16 threads per row, kRows rows per thread.
template <typename T, bool kQuantize, int kRows>
__global__ void __launch_bounds__(256) append_rows_kernel(const AppendParams p) {
  const unsigned total = (unsigned)p.batch * p.tokens * p.heads;
  const int lane = threadIdx.x & 15;
  const unsigned first = blockIdx.x * (16u * kRows) + (threadIdx.x >> 4);
  AppendRow row[kRows];
  Eight<T> x[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    row[i] = append_row(p, first + 16u * i, total);
    if (row[i].live)
      x[i].load(static_cast<const T *>(p.src[row[i].side].data) +
                row_offset(p.src[row[i].side], row[i].b, row[i].h, row[i].t) + lane * 8);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const AppendRow &a = row[i];
    const SharedTensor &dst = p.dst[a.side];
    if constexpr (!kQuantize) {
      if (a.live)
        x[i].store(static_cast<T *>(const_cast<void *>(dst.data)) + row_offset(dst, a.b, a.h, a.pos) + lane * 8);
      continue;
    }
    float f[8];
    if (a.live) {
      x[i].floats(f);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = 0.f;
    }
    float mx = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) mx = fmaxf(mx, finite_abs(f[k]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float sc = row_scale(mx);
    uint2 o;
    o.x = (uint32_t)e4m3x2(__fdiv_rn(f[0], sc), __fdiv_rn(f[1], sc)) |
          ((uint32_t)e4m3x2(__fdiv_rn(f[2], sc), __fdiv_rn(f[3], sc)) << 16);
    o.y = (uint32_t)e4m3x2(__fdiv_rn(f[4], sc), __fdiv_rn(f[5], sc)) |
          ((uint32_t)e4m3x2(__fdiv_rn(f[6], sc), __fdiv_rn(f[7], sc)) << 16);
    if (a.live) {
      *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(const_cast<void *>(dst.data)) +
                                 row_offset(dst, a.b, a.h, a.pos) + lane * 8) = o;
      if (lane == 0)
        static_cast<float *>(const_cast<void *>(p.scale[a.side].data))[row_offset(p.scale[a.side], a.b, a.h, a.pos)] = sc;
    }
  }
}

// Any head width and strides: one warp per row.
template <typename T, bool kQuantize>
__global__ void __launch_bounds__(256) append_any_kernel(const AppendParams p) {
  const unsigned total = (unsigned)p.batch * p.tokens * p.heads;
  const int lane = threadIdx.x & 31;
  const AppendRow a = append_row(p, blockIdx.x * 8u + (threadIdx.x >> 5), total);
  if (!a.live) return;                   // whole warp
  const SharedTensor &src = p.src[a.side], &dst = p.dst[a.side];
  const T *x = static_cast<const T *>(src.data) + row_offset(src, a.b, a.h, a.t);
  const long long to = row_offset(dst, a.b, a.h, a.pos);
  if constexpr (!kQuantize) {
    T *y = static_cast<T *>(const_cast<void *>(dst.data)) + to;
    for (int d = lane; d < p.head_dim; d += 32) y[d * dst.s[3]] = x[d * src.s[3]];
  } else {
    float mx = 0.f;
    for (int d = lane; d < p.head_dim; d += 32) mx = fmaxf(mx, finite_abs(to_f32(x[d * src.s[3]])));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float sc = row_scale(mx);
    uint8_t *y = static_cast<uint8_t *>(const_cast<void *>(dst.data)) + to;
    for (int d = lane; d < p.head_dim; d += 32)
      y[d * dst.s[3]] = (uint8_t)(e4m3x2(__fdiv_rn(to_f32(x[d * src.s[3]]), sc), 0.f) & 0xff);
    if (lane == 0)
      static_cast<float *>(const_cast<void *>(p.scale[a.side].data))[row_offset(p.scale[a.side], a.b, a.h, a.pos)] = sc;
  }
}

template <typename T, bool kQuantize>
cudaError_t append(const AppendParams &p, bool rows128, cudaStream_t stream) {
  const long long rows = 2ll * p.batch * p.tokens * p.heads;
  if (!rows128) {
    append_any_kernel<T, kQuantize><<<(unsigned)((rows + 7) / 8), 256, 0, stream>>>(p);
  } else {
    append_rows_kernel<T, kQuantize, 1><<<(unsigned)((rows + 15) / 16), 256, 0, stream>>>(p);
  }
  return cudaGetLastError();
}

__device__ __forceinline__ float e4m3_value(uint8_t b) {
  __nv_fp8_e4m3 v;
  v.__x = b;
  return static_cast<float>(v);
}

// Any head width and strides: one warp per row of either cache.
template <typename T>
__global__ void __launch_bounds__(256) read_any_kernel(const ReadParams p) {
  const unsigned total = (unsigned)p.batch * p.heads * p.cap;
  unsigned r = blockIdx.x * 8u + (threadIdx.x >> 5);
  if (r >= 2u * total) return;
  const int side = r >= total, lane = threadIdx.x & 31;
  unsigned i = side ? r - total : r;
  const int s = i % p.cap;
  i /= p.cap;
  const int h = i % p.heads, b = i / p.heads;
  const SharedTensor &src = p.src[side], &dst = p.dst[side];
  T *y = static_cast<T *>(const_cast<void *>(dst.data)) + row_offset(dst, b, h, s);
  if (s >= p.lens[b * p.lens_s]) {
    for (int d = lane; d < p.head_dim; d += 32) y[d * dst.s[3]] = from_f32<T>(0.f);
    return;
  }
  const uint8_t *x = static_cast<const uint8_t *>(src.data) + row_offset(src, b, h, s);
  const float sc = static_cast<const float *>(p.scale[side].data)[row_offset(p.scale[side], b, h, s)];
  for (int d = lane; d < p.head_dim; d += 32) y[d * dst.s[3]] = from_f32<T>(e4m3_value(x[d * src.s[3]]) * sc);
}

template <typename T>
cudaError_t read(const ReadParams &p, cudaStream_t stream) {
  const long long rows = 2ll * p.batch * p.heads * p.cap;
  read_any_kernel<T><<<(unsigned)((rows + 7) / 8), 256, 0, stream>>>(p);
  return cudaGetLastError();
}

// rows of 128 elements of `esize` bytes that 16 threads (or 8) can move in
// `align`-byte pieces
bool aligned_rows(const SharedTensor &x, int esize, int align) {
  return x.s[3] == 1 && reinterpret_cast<uintptr_t>(x.data) % align == 0 && x.s[0] * esize % align == 0 &&
         x.s[1] * esize % align == 0 && x.s[2] * esize % align == 0;
}

}  // namespace

cudaError_t launch_append_text(const AppendParams &p, cudaStream_t stream) {
  if ((long long)p.batch * p.tokens * p.heads == 0) return cudaSuccess;
  const int esize = p.dtype == 0 ? 4 : 2;
  bool rows128 = p.head_dim == 128;
  for (int i = 0; i < 2; ++i)
    rows128 = rows128 && aligned_rows(p.src[i], esize, 16) &&
              (p.quantize ? aligned_rows(p.dst[i], 1, 8) : aligned_rows(p.dst[i], esize, 16));
  if (p.quantize) {
    if (p.dtype == 0) return append<float, true>(p, rows128, stream);
    if (p.dtype == 1) return append<__nv_bfloat16, true>(p, rows128, stream);
    return append<__half, true>(p, rows128, stream);
  }
  if (p.dtype == 0) return append<float, false>(p, rows128, stream);
  if (p.dtype == 1) return append<__nv_bfloat16, false>(p, rows128, stream);
  return append<__half, false>(p, rows128, stream);
}

cudaError_t launch_read_text(const ReadParams &p, cudaStream_t stream) {
  if ((long long)p.batch * p.heads * p.cap == 0) return cudaSuccess;
  if (p.dtype == 0) return read<float>(p, stream);
  if (p.dtype == 1) return read<__nv_bfloat16>(p, stream);
  return read<__half>(p, stream);
}

}  // namespace rtk
