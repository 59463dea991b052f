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
// channels take 16-byte accesses; anything else takes the scalar kernels below them.
//
// Measured: 64 x 8 x up to 577 new bf16 tokens appended, 153 MB, in 34.5 us (4.4 TB/s); 64 x 8 x
// 1024 rows read back as fp16, 90 MB in and 268 MB out, in 65 us (5.5 TB/s; a plain fill
// writes at 3.84 TB/s, so it is the writing that bounds it).
#include "common.cuh"
#include "shared.h"

#include <cuda_fp8.h>

#include <type_traits>

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
  // amax / 448 rounded to nearest, as the quotients below (exact remainder down to 2^-126)
  const float r = 1.f / kE4m3Max, q = amax * r;
  return amax > 0.f ? fmaxf(fmaf(-fmaf(q, kE4m3Max, -amax), r, q), 1.17549435e-38f) : 1.f;
}

__device__ __forceinline__ long long row_offset(const SharedTensor &x, int b, int h, int s) {
  return b * x.s[0] + h * x.s[1] + s * x.s[2];
}

// the larger, NaN if either is
__device__ __forceinline__ float larger(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// 16 channels of a row (32 or 64 bytes)
template <typename T>
struct Sixteen {
  static constexpr int kWords = sizeof(T);           // 16-byte words
  uint4 raw[kWords];
  __device__ __forceinline__ void load(const T *src) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) raw[i] = __ldg(reinterpret_cast<const uint4 *>(src) + i);
  }
  __device__ __forceinline__ void store(T *dst) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<uint4 *>(dst)[i] = raw[i];
  }
  // the largest |x|, NaN if there is one (16-bit types two at a time)
  __device__ __forceinline__ float amax() const {
    if constexpr (sizeof(T) == 4) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        m = larger(m, larger(larger(fabsf(__uint_as_float(raw[i].x)), fabsf(__uint_as_float(raw[i].y))),
                             larger(fabsf(__uint_as_float(raw[i].z)), fabsf(__uint_as_float(raw[i].w)))));
      return m;
    } else {
      using T2 = typename std::conditional<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>::type;
      auto h2 = [](uint32_t w) { return __habs2(*reinterpret_cast<const T2 *>(&w)); };
      T2 m = __hmax2_nan(h2(raw[0].x), h2(raw[1].x));
      m = __hmax2_nan(m, __hmax2_nan(h2(raw[0].y), h2(raw[1].y)));
      m = __hmax2_nan(m, __hmax2_nan(h2(raw[0].z), h2(raw[1].z)));
      m = __hmax2_nan(m, __hmax2_nan(h2(raw[0].w), h2(raw[1].w)));
      float lo, hi;
      unpack2<T>(*reinterpret_cast<const uint32_t *>(&m), lo, hi);
      return larger(lo, hi);
    }
  }
  __device__ __forceinline__ void floats(float (&f)[16]) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 4) f[4 * i + k] = __uint_as_float(w[k]);
        else unpack2<T>(w[k], f[8 * i + 2 * k], f[8 * i + 2 * k + 1]);
      }
    }
  }
};

// -(x / s), each rounded to nearest, for two finite numbers and r = 1 / s rounded to nearest:
// with q = x r it is -q - (x - q s) r (Markstein 1990: correctly rounded while the remainder
// x - q s is exact, which s >= 2^-80 grants for every quotient that e4m3 does not round to 0).
// Negated, because then every step is a fused multiply-add of what is there already, and -0
// comes out as what it should be: the sign is put right in the packed bytes.
__device__ __forceinline__ float2 minus_quotient(float2 x, float s, float r) {
  const float2 q = __fmul2_rn(x, make_float2(-r, -r));
  return __ffma2_rn(__ffma2_rn(q, make_float2(s, s), x), make_float2(-r, -r), q);
}

// D = 128: 8 threads per row of 16 channels each, kRows rows per thread.  A CTA takes
// 32 kRows tokens of one head of one question's Keys or Values.  What it costs besides the
// bytes is a dozen instructions a channel (unpacking, the maximum, two to divide, the
// conversion, the row's scale): 16 channels a thread so that the scale and its reciprocal are
// worked out by 8 threads and not by 16, and five CTAs an SM (the 153 MB above: 41 us with one
// quotient at a time and three CTAs, 39 with two, 37 with four CTAs, 34.5 with five).
template <typename T, bool kQuantize, int kRows>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 2 : 5) append_rows_kernel(const AppendParams p, int ctas) {
  const int lane = threadIdx.x & 7;
  const int item = blockIdx.x / ctas, part = blockIdx.x % ctas;
  const int side = item & 1, bh = item >> 1, b = bh / p.heads, h = bh % p.heads;
  const int len = p.lens[b * p.lens_s];
  int count = p.counts != nullptr ? min(p.counts[b * p.counts_s], p.tokens) : p.tokens;
  count = (int)min((long long)count, (long long)p.cap - len);    // tokens below it fit
  if (part * (32 * kRows) >= count) return;
  const SharedTensor &src = p.src[side], &dst = p.dst[side], &scl = p.scale[side];
  const int first = part * (32 * kRows) + (threadIdx.x >> 3);
  const T *from = static_cast<const T *>(src.data) + row_offset(src, b, h, 0) + lane * 16;
  const long long base = row_offset(dst, b, h, 0) + lane * 16;
  Sixteen<T> x[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int t = first + 32 * i;
    if (t < count && t + len >= 0) x[i].load(from + t * src.s[2]);
  }
  const int last = count - ((threadIdx.x & ~31) >> 3);      // of this warp's first row
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (part * (32 * kRows) + 32 * i >= last) break;         // no row of this warp is there
    const int t = first + 32 * i;
    const bool live = t < count && t + len >= 0;
    const long long to = base + (long long)(len + t) * dst.s[2];
    if constexpr (!kQuantize) {
      if (live) x[i].store(static_cast<T *>(const_cast<void *>(dst.data)) + to);
      continue;
    }
    if (!live) {
#pragma unroll
      for (int k = 0; k < Sixteen<T>::kWords; ++k) x[i].raw[k] = make_uint4(0, 0, 0, 0);
    }
    float f[16];
    x[i].floats(f);
    float mx = x[i].amax();
    const bool finite = mx < INFINITY;
    if (!finite) {
      mx = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) mx = fmaxf(mx, finite_abs(f[k]));
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float sc = row_scale(mx);
    uint32_t flip = 0u;
    if (finite && sc >= 8.2718061e-25f) {
      const float r = __frcp_rn(sc);
      flip = 0x80808080u;
#pragma unroll
      for (int k = 0; k < 16; k += 2) {
        const float2 y = minus_quotient(make_float2(f[k], f[k + 1]), sc, r);
        f[k] = y.x;
        f[k + 1] = y.y;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) f[k] = __fdiv_rn(f[k], sc);
    }
    uint32_t o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      o[k] = ((uint32_t)e4m3x2(f[4 * k], f[4 * k + 1]) | ((uint32_t)e4m3x2(f[4 * k + 2], f[4 * k + 3]) << 16)) ^ flip;
    if (live) {
      *reinterpret_cast<uint4 *>(static_cast<uint8_t *>(const_cast<void *>(dst.data)) + to) =
          make_uint4(o[0], o[1], o[2], o[3]);
      if (lane == 0)
        static_cast<float *>(const_cast<void *>(scl.data))[row_offset(scl, b, h, 0) + (long long)(len + t) * scl.s[2]] = sc;
    }
  }
}

// Any head width and strides: one warp per row.
template <typename T, bool kQuantize>
__global__ void __launch_bounds__(256) append_any_kernel(const AppendParams p) {
  const unsigned total = (unsigned)p.batch * p.tokens * p.heads;
  const int lane = threadIdx.x & 31;
  const unsigned r = blockIdx.x * 8u + (threadIdx.x >> 5);
  if (r >= 2u * total) return;           // whole warp, here and below
  const int side = r >= total;
  unsigned i = side ? r - total : r;
  const int h = i % p.heads;
  i /= p.heads;
  const int t = i % p.tokens, b = i / p.tokens, pos = p.lens[b * p.lens_s] + t;
  if (t >= (p.counts != nullptr ? p.counts[b * p.counts_s] : p.tokens) || pos < 0 || pos >= p.cap) return;
  const SharedTensor &src = p.src[side], &dst = p.dst[side];
  const T *x = static_cast<const T *>(src.data) + row_offset(src, b, h, t);
  const long long to = row_offset(dst, b, h, pos);
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
      static_cast<float *>(const_cast<void *>(p.scale[side].data))[row_offset(p.scale[side], b, h, pos)] = sc;
  }
}

template <typename T, bool kQuantize>
cudaError_t append(const AppendParams &p, bool rows128, cudaStream_t stream) {
  const long long rows = 2ll * p.batch * p.heads * p.tokens;
  const int items = 2 * p.batch * p.heads;
  if (!rows128) {
    append_any_kernel<T, kQuantize><<<(unsigned)((rows + 7) / 8), 256, 0, stream>>>(p);
  } else if (rows <= 32 * 1024) {
    // few rows: spread them over the SMs (one token of 8 questions: 2.2 us, 3.1 with four)
    const int ctas = (p.tokens + 31) / 32;
    append_rows_kernel<T, kQuantize, 1><<<items * ctas, 256, 0, stream>>>(p, ctas);
  } else {
    // many: three rows of a thread in flight (the 153 MB: 37 us with four, 39 with two)
    const int ctas = (p.tokens + 95) / 96;
    append_rows_kernel<T, kQuantize, 3><<<items * ctas, 256, 0, stream>>>(p, ctas);
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

// D = 128: 8 threads per row (16 bytes each), 32 tokens of one (question, head) of either
// cache per CTA.
template <typename T>
__global__ void __launch_bounds__(256) read_rows_kernel(const ReadParams p, int ctas) {
  const int item = blockIdx.x / ctas, part = blockIdx.x % ctas;
  const int side = item & 1, bh = item >> 1, b = bh / p.heads, h = bh % p.heads;
  const int lane = threadIdx.x & 7, s = part * 32 + (threadIdx.x >> 3);
  const int len = p.lens[b * p.lens_s];
  const SharedTensor &src = p.src[side], &dst = p.dst[side], &scl = p.scale[side];
  const uint8_t *x = static_cast<const uint8_t *>(src.data) + row_offset(src, b, h, 0) + lane * 16;
  const float *sc = static_cast<const float *>(scl.data) + row_offset(scl, b, h, 0);
  T *y = static_cast<T *>(const_cast<void *>(dst.data)) + row_offset(dst, b, h, 0) + lane * 16;
  if (s >= p.cap) return;
  const uint4 raw = s < len ? __ldg(reinterpret_cast<const uint4 *>(x + s * src.s[2])) : make_uint4(0, 0, 0, 0);
  const float scale = s < len ? __ldg(sc + s * scl.s[2]) : 0.f;
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  float f[16];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    uint32_t hh;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hh) : "h"((uint16_t)(w[k >> 1] >> (16 * (k & 1)))));
    unpack2<__half>(hh, f[2 * k], f[2 * k + 1]);
    f[2 * k] *= scale;
    f[2 * k + 1] *= scale;
  }
  uint4 *to = reinterpret_cast<uint4 *>(y + s * dst.s[2]);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      to[k] = make_uint4(__float_as_uint(f[4 * k]), __float_as_uint(f[4 * k + 1]), __float_as_uint(f[4 * k + 2]),
                         __float_as_uint(f[4 * k + 3]));
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      __stcs(to + k, make_uint4(pack2<T>(f[8 * k], f[8 * k + 1]), pack2<T>(f[8 * k + 2], f[8 * k + 3]),
                                pack2<T>(f[8 * k + 4], f[8 * k + 5]), pack2<T>(f[8 * k + 6], f[8 * k + 7])));
  }
}

template <typename T>
cudaError_t read(const ReadParams &p, bool rows128, cudaStream_t stream) {
  const long long rows = 2ll * p.batch * p.heads * p.cap;
  const int items = 2 * p.batch * p.heads;
  if (!rows128) {
    read_any_kernel<T><<<(unsigned)((rows + 7) / 8), 256, 0, stream>>>(p);
  } else {
    const int ctas = (p.cap + 31) / 32;
    read_rows_kernel<T><<<items * ctas, 256, 0, stream>>>(p, ctas);
  }
  return cudaGetLastError();
}

// rows of 128 elements of `esize` bytes that threads can move 16 bytes at a time: the strides of
// dimensions with more than one entry are whole pieces
bool aligned_rows(const SharedTensor &x, int batch, int heads, int rows, int esize) {
  const int entries[3] = {batch, heads, rows};
  for (int i = 0; i < 3; ++i)
    if (entries[i] > 1 && x.s[i] * esize % 16 != 0) return false;
  return x.s[3] == 1 && reinterpret_cast<uintptr_t>(x.data) % 16 == 0;
}

}  // namespace

cudaError_t launch_append_text(const AppendParams &p, cudaStream_t stream) {
  if ((long long)p.batch * p.tokens * p.heads == 0) return cudaSuccess;
  const int esize = p.dtype == 0 ? 4 : 2;
  bool rows128 = p.head_dim == 128;
  for (int i = 0; i < 2; ++i)
    rows128 = rows128 && aligned_rows(p.src[i], p.batch, p.heads, p.tokens, esize) &&
              aligned_rows(p.dst[i], p.batch, p.heads, p.cap, p.quantize ? 1 : esize);
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
  const int esize = p.dtype == 0 ? 4 : 2;
  bool rows128 = p.head_dim == 128;
  for (int i = 0; i < 2; ++i)
    rows128 = rows128 && aligned_rows(p.src[i], p.batch, p.heads, p.cap, 1) &&
              aligned_rows(p.dst[i], p.batch, p.heads, p.cap, esize);
  if (p.dtype == 0) return read<float>(p, rows128, stream);
  if (p.dtype == 1) return read<__nv_bfloat16>(p, rows128, stream);
  return read<__half>(p, rows128, stream);
}

}  // namespace rtk
