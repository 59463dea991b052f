// Shared-prefix attention, the text part: each question's T tokens and G heads of a
// KV head (rows = T G, few) over that question's own text cache.
//
//   x_s = c s_k[s] (q . k[s]),  c = log2(e) / sqrt(D);   O = sum 2^(x_s - m) s_v[s] v[s]
// (s_k, s_v: the scales of 8-bit rows, 1 otherwise), over the tokens that query t sees.
//
// A question's text belongs to it alone: its bytes are read once for a handful of rows.  The
// work is cut into (question, KV head, chunk of tokens), so that bytes stay in flight on every
// SM, and m16n8k16 MMAs take the rows as M: S = Q . K^T, and O += P . V with P straight out of
// S's registers.  m follows the maximum lazily (it moves when a maximum is more than 2^8 above
// it).  Two kernels:
//
// - The warps split the rows, 16 each (64 of a CTA), and share tiles of 32 tokens through one
//   cp.async ring; an 8-bit tile is converted to 16 bits in shared memory once for all of them.
// - 8-bit text of at most 16 rows: the warps split the tokens, blocks of 32 in rings of their
//   own (no CTA-wide barrier in the loop), convert in registers, and join at the end.
//
// Measured (the whole attention of a step, prefix of 1064 tokens): 8-bit, 64 questions, 8 heads
// of 8 rows, up to 4096 tokens 105 us with split tokens, 171 with split rows; 256 questions, 8
// heads of 4, 512 tokens 75.7 and 103; 64, 4 heads of 14, 1024 tokens 37.4 and 44.7.  16-bit text
// always takes split rows: no conversion to share, and less to join at the end (when both took
// it, with one part of P, 112.8 us by rows and 113.8 by tokens for the first of these, 75.5 and
// 80.0 for the second).  The kernels alone: 64 questions, 8 heads of 64 rows, up to 1001 tokens of
// 8 bits 72 us; 64, 4 heads of 35 rows, 512 tokens 21; 64, 8 heads of 8 rows, 4096 tokens 91 us
// of 8 bits, 105 of 16.
//
// What bounds it: with 16-bit text and many questions HBM and the second part of P (537 MB in 105
// us, 5.1 TB/s); with 8-bit text the conversions (277 MB in 91 us) and, for many rows, the MMAs'
// issue; with few questions the latency of a chunk.
//
// 8-bit text: e4m3 is exact in f16 and in bf16.  S runs in the queries' type, a token's Key
// scale multiplies its logit.  P . V runs in bf16, which has fp32's range: a token's Value scale
// multiplies its weight, and scales of any ratio may meet in one row.
// In registers: ldmatrix of Key bytes gives lane (g, j) bytes 4j .. 4j+3 of token g: the MMA's
// k index runs over a 16-channel group in the order 0 1 4 5 8 9 12 13 2 3 6 7 10 11 14 15, and
// the queries are stored in that order.  ldmatrix.trans of Value bytes pairs two tokens' bytes
// of channels (2g, 2g+1): one byte permute separates them into B fragments of an "even" and
// an "odd" n-tile.  P is taken in two 16-bit parts, as the prefix kernel's; l sums it unrounded.
//
// Tokens past the length are zero-filled on the way in (cp.async reads nothing there).  The last
// T - 1 tokens within it are seen by some rows only: their weight is 0 in the others, but 0 times
// a Value that is not finite is NaN.  Such Values are taken out of their tile, and the rows that
// do see one (a row that sees a token sees all before it) get NaN in its channel at the end.
//
// The kernels may run beside the prefix kernel launched before (they need nothing of it); one
// CTA waits for that one before it ends, so that the join, which waits for this kernel to
// end, finds both done.  (Where every CTA waited, the first of them held their SMs.)
#include <type_traits>

#include "common.cuh"
#include "shared.h"

namespace rtk {
namespace {

constexpr int kWarps = 4;
constexpr float kLazy = 8.f;

// ---- the warps split the tokens: 8-bit text of at most 16 rows
struct TextSmem {
  static constexpr int kTok = 32;                          // tokens of a block
  static constexpr int kRow = 128;                         // bytes of a token's Key (or Value)
  static constexpr int kScales = 2 * kTok * kRow;          // the tokens' Key scales, Value scales
  static constexpr int kStage = kScales + 2 * kTok * 4;           // 8 KB and the scales
  static constexpr int kStages = 2;
  static constexpr int kQ = 0;                             // 16 rows of 256 bytes
  static constexpr int kRing = kQ + 4096;
  static constexpr int kBytes = kRing + kWarps * kStages * kStage;
  // after the loop: O [4][16][128] and (m, l) [4][16], over the ring
  static constexpr int kMerge = kWarps * 16 * (128 + 2) * 4;
  static_assert(kMerge <= kWarps * kStages * kStage, "merge area");
};

// 16-byte chunk c of row r, rows of kRow bytes: chunks XORed with the row spread the
// eight rows of an ldmatrix over the banks
template <int kRow>
__device__ __forceinline__ uint32_t at(int r, int c) {
  return (uint32_t)(r * kRow + ((c ^ (r & 7)) << 4));
}

// 4-byte global -> shared copy; zero where `in` is false
__device__ __forceinline__ void cp_async_4_zfill(void *dst, const void *src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 4 : 0) : "memory");
}

// Chunk c of this lane's row of an ldmatrix, given the address of its chunk `odd` (0 or 1)
// there: c = even + odd, and XOR with an even chunk number is one instruction (rows start
// at multiples of 256 bytes).
__device__ __forceinline__ uint32_t even(uint32_t lane_addr, int even_chunk) { return lane_addr ^ (even_chunk << 4); }

__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}

__device__ __forceinline__ uint32_t e4m3x2_bf16x2(uint16_t v) {
  float lo, hi;
  unpack2<__half>(e4m3x2_f16x2(v), lo, hi);
  return pack2<__nv_bfloat16>(lo, hi);
}

template <typename T>
__device__ __forceinline__ uint32_t e4m3x2_16(uint16_t v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return e4m3x2_bf16x2(v);
  else return e4m3x2_f16x2(v);
}

// Two weights as 16-bit parts: the nearest, and the nearest to what that leaves.
template <typename M>
__device__ __forceinline__ void two_parts(float w0, float w1, uint32_t &hi, uint32_t &lo) {
  float h0, h1;
  hi = pack2<M>(w0, w1);
  unpack2<M>(hi, h0, h1);
  lo = pack2<M>(w0 - h0, w1 - h1);
}

// Whether a 16-byte piece holds infinities or NaN: an exponent of ones (e4m3: all of 0x7f)
// carries into the sign's place.
template <typename M>
__device__ __forceinline__ bool not_finite(const uint4 &v) {
  constexpr bool k8 = sizeof(M) == 1;
  constexpr uint32_t kUnit = k8 ? 0x01010101u : std::is_same<M, __nv_bfloat16>::value ? 0x00800080u : 0x04000400u;
  constexpr uint32_t kSign = k8 ? 0x80808080u : 0x80008000u;
  auto carry = [](uint32_t w) { return (w & ~kSign) + kUnit; };
  return ((carry(v.x) | carry(v.y) | carry(v.z) | carry(v.w)) & kSign) != 0;
}

constexpr int kNoToken = 0x7fffffff;

// Values (M, or e4m3 bytes) of tokens [s0, s1) of a tile that are not finite become 0; the first such
// token of a channel is left in apart_s.  By a whole warp; warps that share a tile may do the
// same at once.
template <typename M>
__device__ __noinline__ void take_apart(unsigned char *tile, int s0, int s1, int first, int *apart_s) {
  constexpr int kRow = 128 * sizeof(M), kPieces = kRow / 16, kEach = 16 / sizeof(M);
  using Bits = typename std::conditional<sizeof(M) == 1, unsigned char, unsigned short>::type;
  constexpr unsigned kTop = sizeof(M) == 1 ? 0x7fu : std::is_same<M, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  const int lane = threadIdx.x & 31;
  for (int s = s0; s < s1; ++s) {
    if (lane >= kPieces) continue;
    Bits *x = reinterpret_cast<Bits *>(tile + at<kRow>(s, lane));
    for (int k = 0; k < kEach; ++k)
      if ((x[k] & kTop) == kTop) {
        atomicMin(&apart_s[lane * kEach + k], first + s);
        x[k] = 0;
      }
  }
  __syncwarp();
}

// Whether tokens [s0, s1) of a tile hold a Value that is not finite; the whole warp asks.
template <typename M>
__device__ __forceinline__ bool any_not_finite(const unsigned char *tile, int s0, int s1) {
  constexpr int kRow = 128 * sizeof(M), kPieces = kRow / 16;
  const int lane = threadIdx.x & 31;
  bool any = false;
  for (int s = s0 + lane / kPieces; s < s1; s += 32 / kPieces)
    any |= not_finite<M>(*reinterpret_cast<const uint4 *>(tile + at<kRow>(s, lane % kPieces)));
  return __any_sync(0xffffffffu, any);
}

// The same for Value scales: vscale[n][k] is that of token 8 n + 2 j4 + k, `scales` the tile's in shared memory.
__device__ __forceinline__ bool scales_apart(const unsigned char *scales, float (&vscale)[4][2], int s0, int s1, int first,
                                             int *apart_s) {
  const int lane = threadIdx.x & 31;
  const uint32_t bad = __ballot_sync(0xffffffffu, lane >= s0 && lane < s1 && !isfinite(reinterpret_cast<const float *>(scales)[lane]));
  if (bad == 0) return false;
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if ((bad >> (8 * n + 2 * (lane & 3) + k)) & 1u) vscale[n][k] = 0.f;
  for (int c = lane; c < 128; c += 32) atomicMin(&apart_s[c], first + __ffs(bad) - 1);
  return true;
}

// The kernel ends after the one before it.
__device__ __forceinline__ void end_after_previous() {
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) wait_for_previous();
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32, 3) shared_text_kernel(const TextParams p) {
  using L = TextSmem;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ int apart_s[128];                       // per channel: the first token taken apart
  launch_dependents();
  const SharedParams &a = p.s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, j4 = lane & 3;
  const int chunk = blockIdx.y, bh = blockIdx.x;
  apart_s[threadIdx.x] = kNoToken;
  const int b = bh / a.kv_heads, h = bh % a.kv_heads;
  const int len = min(max(a.lens[b * a.lens_s], 0), a.cap);
  const int t0 = chunk * p.chunk;
  if (t0 >= len) {
    end_after_previous();
    return;
  }
  const int t1 = min(len, t0 + p.chunk);
  const int blocks = (t1 - t0 + L::kTok - 1) / L::kTok;

  // this warp's ring
  unsigned char *ring = smem + L::kRing + warp * L::kStages * L::kStage;
  const unsigned char *kbase = static_cast<const unsigned char *>(a.kt.data) + b * a.kt.s[0] + h * a.kt.s[1];
  const unsigned char *vbase = static_cast<const unsigned char *>(a.vt.data) + b * a.vt.s[0] + h * a.vt.s[1];
  const long long ks = a.kt.s[2], vs = a.vt.s[2];
  const float *ksc = static_cast<const float *>(a.ksc.data) + b * a.ksc.s[0] + h * a.ksc.s[1];
  const float *vsc = static_cast<const float *>(a.vsc.data) + b * a.vsc.s[0] + h * a.vsc.s[1];
  auto fetch = [&](int blk, int stage) {
    unsigned char *dst = ring + stage * L::kStage;
    constexpr int kChunks = L::kRow / 16;
    const int first = t0 + blk * L::kTok;
#pragma unroll
    for (int e = 0; e < L::kTok * kChunks / 32; ++e) {
      const int i = e * 32 + lane, r = i / kChunks, c = i % kChunks;
      const int tok = first + r;
      const bool in = tok < t1;
      cp_async_16_zfill(dst + at<L::kRow>(r, c), kbase + (in ? tok * ks + c * 16 : 0), in ? 16 : 0);
      cp_async_16_zfill(dst + L::kTok * L::kRow + at<L::kRow>(r, c), vbase + (in ? tok * vs + c * 16 : 0), in ? 16 : 0);
    }
    // lane = token of the block
    const bool in = first + lane < t1;
    cp_async_4_zfill(dst + L::kScales + lane * 4, ksc + (in ? (first + lane) * a.ksc.s[2] : 0), in);
    cp_async_4_zfill(dst + L::kScales + 128 + lane * 4, vsc + (in ? (first + lane) * a.vsc.s[2] : 0), in);
  };
#pragma unroll
  for (int i = 0; i < L::kStages - 1; ++i) {
    if (warp + kWarps * i < blocks) fetch(warp + kWarps * i, i);
    cp_async_commit();
  }

  // queries: 16 rows x 128 channels
  uint2 qv[4];                                       // all in flight at once
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = warp + kWarps * k;
    qv[k] = make_uint2(0, 0);                        // channels 4 lane .. 4 lane + 3
    if (r < p.rows) {
      const int t = r / a.groups, gh = r % a.groups;
      qv[k] = __ldg(reinterpret_cast<const uint2 *>(static_cast<const T *>(a.q.data) + b * a.q.s[0] + t * a.q.s[1] +
                                                    (h * a.groups + gh) * a.q.s[2] + lane * 4));
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int e = warp + kWarps * k;
    // channels 4 jj .. 4 jj + 3 of a 16-channel group go to positions 2 jj, 2 jj + 1 and
    // 2 jj + 8, 2 jj + 9 (lane = 4 * group + jj)
    const int grp = lane >> 2, jj = lane & 3;
    const uint32_t q0 = smem_u32(smem + L::kQ);
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(q0 + at<256>(e, 2 * grp) + jj * 4), "r"(qv[k].x) : "memory");
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(q0 + at<256>(e, 2 * grp + 1) + jj * 4), "r"(qv[k].y) : "memory");
  }
  __syncthreads();

  // tokens that the query rows of this lane (g and g + 8) see
  int limit[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = g + 8 * i;
    limit[i] = r < p.rows ? len - (a.tokens - 1 - r / a.groups) : 0;
  }
  const int all_see = len - (a.tokens - 1);          // every row sees tokens below this

  float m[2], l[2], acc[16][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
#pragma unroll
  for (int n = 0; n < 16; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  const uint32_t q_lane = smem_u32(smem + L::kQ) + at<256>(lane & 15, lane >> 4);

  int stage = 0;
  bool apart = false;
  for (int blk = warp; blk < blocks; blk += kWarps) {
    const int first = t0 + blk * L::kTok;
    constexpr int kNT = L::kTok / 8;                 // n-tiles of 8 tokens
    float kscale[kNT][2], vscale[kNT][2];
    {
      const int next = blk + kWarps * (L::kStages - 1);
      int st2 = stage + L::kStages - 1;
      if (st2 >= L::kStages) st2 -= L::kStages;
      if (next < blocks) fetch(next, st2);
      cp_async_commit();
    }
    cp_async_wait_group<L::kStages - 1>();
    __syncwarp();
    const uint32_t k_addr = smem_u32(ring + stage * L::kStage), v_addr = k_addr + L::kTok * L::kRow;
    const unsigned char *sc = ring + stage * L::kStage + L::kScales;
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      const float2 k2 = *reinterpret_cast<const float2 *>(sc + (n * 8 + 2 * j4) * 4);
      const float2 v2 = *reinterpret_cast<const float2 *>(sc + 128 + (n * 8 + 2 * j4) * 4);
      kscale[n][0] = k2.x; kscale[n][1] = k2.y;
      vscale[n][0] = v2.x; vscale[n][1] = v2.y;
    }
    if (all_see < min(t1, first + L::kTok)) {      // tokens that some rows do not see
      const int s0 = max(all_see - first, 0), s1 = min(t1 - first, L::kTok);
      unsigned char *v = ring + stage * L::kStage + L::kTok * L::kRow;
      if (any_not_finite<unsigned char>(v, s0, s1)) {
        take_apart<unsigned char>(v, s0, s1, first, apart_s);
        apart = true;
      }
      apart |= scales_apart(sc + 128, vscale, s0, s1, first, apart_s);
    }
    float s[kNT][4];
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {                  // 16 channels
      uint32_t qa[4];
      ldmatrix_x4(even(q_lane, 2 * k), qa[0], qa[1], qa[2], qa[3]);
      // four n-tiles of 8 tokens, the 16-byte chunk k of each
      uint32_t r[4];
      ldmatrix_x4(k_addr + at<128>(lane, k), r[0], r[1], r[2], r[3]);
#pragma unroll
      for (int n = 0; n < 4; ++n)
        mma_16816<T>(s[n], qa, e4m3x2_16<T>((uint16_t)(r[n] & 0xffffu)), e4m3x2_16<T>((uint16_t)(r[n] >> 16)));
    }
    // logits but for c; unseen tokens weigh nothing
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] *= kscale[n][i & 1];
    if (first + L::kTok > all_see) {
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (first + n * 8 + 2 * j4 + (i & 1) >= limit[i >> 1]) s[n][i] = -INFINITY;
    }
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx[i >> 1] = fmaxf(mx[i >> 1], s[n][i]);
    // base-2 maxima of the rows; O and l move to a new one only when it is more than 2^8
    // above the one in use
    bool grow[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2)) * a.scale_log2;
      grow[i] = mx[i] > m[i] + kLazy;          // from -inf: whenever there is a maximum
    }
    if (__any_sync(0xffffffffu, grow[0] || grow[1])) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float f = grow[i] ? fast_exp2(m[i] - mx[i]) : 1.f;      // nothing yet: 2^-inf = 0
        if (grow[i]) m[i] = mx[i];
        l[i] *= f;
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          acc[n][2 * i] *= f;
          acc[n][2 * i + 1] *= f;
        }
      }
    }
    const float base[2] = {m[0] > -INFINITY ? m[0] : 0.f, m[1] > -INFINITY ? m[1] : 0.f};
    uint32_t pa[kNT][2], pl[kNT][2];               // weights of rows g, g + 8
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float w0 = fast_exp2(fmaf(s[n][2 * i], a.scale_log2, -base[i]));
        const float w1 = fast_exp2(fmaf(s[n][2 * i + 1], a.scale_log2, -base[i]));
        l[i] += w0 + w1;
        two_parts<__nv_bfloat16>(w0 * vscale[n][0], w1 * vscale[n][1], pa[n][i], pl[n][i]);
      }
#pragma unroll
    for (int kk = 0; kk < kNT / 2; ++kk) {         // 16 tokens
      const uint32_t pf[4] = {pa[2 * kk][0], pa[2 * kk][1], pa[2 * kk + 1][0], pa[2 * kk + 1][1]};
      const uint32_t pg[4] = {pl[2 * kk][0], pl[2 * kk][1], pl[2 * kk + 1][0], pl[2 * kk + 1][1]};
#pragma unroll
      for (int c = 0; c < 8; c += 2) {           // two 16-byte chunks of channels
        uint32_t r[4];
        ldmatrix_x4_trans(v_addr + at<128>(kk * 16 + (lane & 15), c + (lane >> 4)), r[0], r[1], r[2], r[3]);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t lo = __byte_perm(r[2 * q], 0, 0x3120), hi = __byte_perm(r[2 * q + 1], 0, 0x3120);
#pragma unroll
          for (int odd = 0; odd < 2; ++odd) {
            const uint32_t b0 = e4m3x2_bf16x2((uint16_t)(lo >> (16 * odd))), b1 = e4m3x2_bf16x2((uint16_t)(hi >> (16 * odd)));
            mma_16816<__nv_bfloat16>(acc[2 * (c + q) + odd], pf, b0, b1);
            mma_16816<__nv_bfloat16>(acc[2 * (c + q) + odd], pg, b0, b1);
          }
        }
      }
    }
    __syncwarp();
    if (++stage == L::kStages) stage = 0;
  }
  cp_async_wait_all();
  const bool any_apart = __syncthreads_or(apart);    // every warp is done with its ring

  // join the warps, in warp order
  float *o_s = reinterpret_cast<float *>(smem + L::kRing);
  float2 *ml_s = reinterpret_cast<float2 *>(o_s + kWarps * 16 * 128);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float ll = l[i];
    ll += __shfl_xor_sync(0xffffffffu, ll, 1);
    ll += __shfl_xor_sync(0xffffffffu, ll, 2);
    const int e = g + 8 * i;
    if (j4 == 0) ml_s[warp * 16 + e] = make_float2(m[i], ll);
    if (any_apart) {
#pragma unroll
      for (int c = 0; c < 8; ++c)                    // acc[2 c + odd][2 i + k] is channel 16 c + 4 j4 + 2 k + odd
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (limit[i] > apart_s[16 * c + 4 * j4 + k]) acc[2 * c + (k & 1)][2 * i + (k >> 1)] = NAN;
    }
    float *row = o_s + (warp * 16 + e) * 128;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      *reinterpret_cast<float4 *>(row + 16 * c + 4 * j4) =
          make_float4(acc[2 * c][2 * i], acc[2 * c + 1][2 * i], acc[2 * c][2 * i + 1], acc[2 * c + 1][2 * i + 1]);
  }
  __syncthreads();
  // the rows' factors of each warp's partial, over the warps' own (m, l)
  const int rows = p.rows;                           // at most 16
  const long long slot = (long long)bh * p.chunks + chunk;
  if ((int)threadIdx.x < rows) {
    const int e = threadIdx.x;
    float2 st[kWarps];
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      st[w] = ml_s[w * 16 + e];
      mm = fmaxf(mm, st[w].x);
    }
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = st[w].x > -INFINITY ? fast_exp2(st[w].x - mm) : -1.f;    // < 0: saw nothing (its sum is 0)
      ll = fmaf(st[w].y, f, ll);
      ml_s[w * 16 + e].x = f;
    }
    reinterpret_cast<float2 *>(p.ml)[slot * p.rows + e] = make_float2(isnan(ll) ? ll : mm, ll);
  }
  __syncthreads();
  float4 *out = reinterpret_cast<float4 *>(p.acc) + slot * 32 * p.rows;
  for (int i = threadIdx.x; i < rows * 32; i += 32 * kWarps) {
    const int c4 = i / rows, e = i - c4 * rows;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ml_s[w * 16 + e].x;
      if (f < 0.f) continue;                         // its O may be anything
      const float4 v = *reinterpret_cast<const float4 *>(o_s + (w * 16 + e) * 128 + c4 * 4);
      o.x = fmaf(v.x, f, o.x);
      o.y = fmaf(v.y, f, o.y);
      o.z = fmaf(v.z, f, o.z);
      o.w = fmaf(v.w, f, o.w);
    }
    out[(long long)c4 * p.rows + e] = o;
  }
  end_after_previous();
}

// ---- the warps split the rows
template <bool FP8>
struct RowsSmem {
  static constexpr int kTok = 32;
  static constexpr int kScales = 2 * kTok * (FP8 ? 128 : 256);    // after a tile's Keys and Values as stored
  static constexpr int kRaw = kScales + (FP8 ? 2 * kTok * 4 : 0);
  static constexpr int kStages = 3;
  static constexpr int kQ = 0;                                    // 64 rows of 256 bytes
  static constexpr int kTile = kQ + kWarps * 4096;                // FP8: the tile, Keys in the queries' type, Values as bf16
  static constexpr int kRing = kTile + (FP8 ? 2 * kTok * 256 : 0);
  static constexpr int kBytes = kRing + kStages * kRaw;
};

template <typename T, bool FP8>
__global__ void __launch_bounds__(kWarps * 32, 3) shared_text_rows_kernel(const TextParams p) {
  using L = RowsSmem<FP8>;
  using MV = typename std::conditional<FP8, __nv_bfloat16, T>::type;     // operand type of P . V (of S: T)
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ int apart_s[128];                       // per channel: the first token taken apart
  launch_dependents();
  const SharedParams &a = p.s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, j4 = lane & 3;
  apart_s[threadIdx.x] = kNoToken;
  const int chunk = blockIdx.y, bh = blockIdx.x, row0 = blockIdx.z * 64 + warp * 16;
  const int b = bh / a.kv_heads, h = bh % a.kv_heads;
  const int len = min(max(a.lens[b * a.lens_s], 0), a.cap);
  const int t0 = chunk * p.chunk;
  if (t0 >= len) {
    end_after_previous();
    return;
  }
  const int t1 = min(len, t0 + p.chunk);
  const int tiles = (t1 - t0 + L::kTok - 1) / L::kTok;
  constexpr int kEsize = FP8 ? 1 : 2, kRowBytes = 128 * kEsize, kChunks = kRowBytes / 16;
  const unsigned char *kbase = static_cast<const unsigned char *>(a.kt.data) + (b * a.kt.s[0] + h * a.kt.s[1]) * kEsize;
  const unsigned char *vbase = static_cast<const unsigned char *>(a.vt.data) + (b * a.vt.s[0] + h * a.vt.s[1]) * kEsize;
  const long long ks = a.kt.s[2] * kEsize, vs = a.vt.s[2] * kEsize;
  const float *ksc = FP8 ? static_cast<const float *>(a.ksc.data) + b * a.ksc.s[0] + h * a.ksc.s[1] : nullptr;
  const float *vsc = FP8 ? static_cast<const float *>(a.vsc.data) + b * a.vsc.s[0] + h * a.vsc.s[1] : nullptr;
  // this thread's first row of a tile and its 16 bytes of it; further rows kRowStep apart
  constexpr int kRowStep = 32 * kWarps / kChunks, kRows = L::kTok / kRowStep;
  const int my_row = threadIdx.x / kChunks, my_chunk = threadIdx.x % kChunks;
  const unsigned char *kp = kbase + (t0 + my_row) * ks + my_chunk * 16, *vp = vbase + (t0 + my_row) * vs + my_chunk * 16;
  int fetched = 0;                                   // tiles asked for so far, one after another
  uint32_t fetch_stage = 0;
  auto fetch = [&] {
    unsigned char *dst = smem + L::kRing + fetch_stage * L::kRaw;
    const int first = t0 + fetched * L::kTok;
#pragma unroll
    for (int e = 0; e < kRows; ++e) {
      const int r = my_row + e * kRowStep;
      const bool in = first + r < t1;
      cp_async_16_zfill(dst + at<kRowBytes>(r, my_chunk), in ? kp + e * kRowStep * ks : kbase, in ? 16 : 0);
      cp_async_16_zfill(dst + L::kTok * kRowBytes + at<kRowBytes>(r, my_chunk), in ? vp + e * kRowStep * vs : vbase, in ? 16 : 0);
    }
    if (FP8 && warp < 2) {                           // lane = token of the tile
      const bool in = first + lane < t1;
      cp_async_4_zfill(dst + L::kScales + warp * 128 + lane * 4,
                       warp == 0 ? ksc + (in ? (first + lane) * a.ksc.s[2] : 0) : vsc + (in ? (first + lane) * a.vsc.s[2] : 0),
                       in);
    }
    kp += L::kTok * ks;
    vp += L::kTok * vs;
    ++fetched;
    if (++fetch_stage == (uint32_t)L::kStages) fetch_stage = 0;
  };
#pragma unroll
  for (int i = 0; i < L::kStages - 1; ++i) {
    if (i < tiles) fetch();
    cp_async_commit();
  }
  // this warp's 16 queries
  uint2 qv[16];                                      // all in flight at once
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int r = row0 + e;
    qv[e] = make_uint2(0, 0);                        // channels 4 lane .. 4 lane + 3
    if (r < p.rows) {
      const int t = r / a.groups, gh = r % a.groups;
      qv[e] = __ldg(reinterpret_cast<const uint2 *>(static_cast<const T *>(a.q.data) + b * a.q.s[0] + t * a.q.s[1] +
                                                    (h * a.groups + gh) * a.q.s[2] + lane * 4));
    }
  }
#pragma unroll
  for (int e = 0; e < 16; ++e)
    *reinterpret_cast<uint2 *>(smem + L::kQ + at<256>(warp * 16 + e, lane >> 1) + (lane & 1) * 8) = qv[e];
  __syncwarp();
  const bool busy = row0 < p.rows;
  int limit[2];
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, acc[16][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = row0 + g + 8 * i;
    limit[i] = r < p.rows ? len - (a.tokens - 1 - r / a.groups) : 0;
  }
#pragma unroll
  for (int n = 0; n < 16; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  const int all_see = len - (a.tokens - 1);          // every row sees tokens below this
  const uint32_t q_lane = smem_u32(smem + L::kQ) + at<256>(warp * 16 + (lane & 15), lane >> 4);
  const uint32_t k_at = at<256>((lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1), v_at = at<256>(lane & 15, lane >> 4);

  bool apart = false;
  for (int tile = 0; tile < tiles; ++tile) {
    const int first = t0 + tile * L::kTok;
    constexpr int kNT = 4;
    float kscale[kNT][2], vscale[kNT][2];
    cp_async_wait_group<L::kStages - 2>();
    __syncthreads();                                 // the tile has landed; the one before is done with
    if (fetched < tiles) fetch();
    cp_async_commit();
    uint32_t k_addr, v_addr;
    const unsigned char *raw = smem + L::kRing + tile % L::kStages * L::kRaw;
    if constexpr (FP8) {
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        const float2 k2 = *reinterpret_cast<const float2 *>(raw + L::kScales + (n * 8 + 2 * j4) * 4);
        const float2 v2 = *reinterpret_cast<const float2 *>(raw + L::kScales + 128 + (n * 8 + 2 * j4) * 4);
        kscale[n][0] = k2.x; kscale[n][1] = k2.y;
        vscale[n][0] = v2.x; vscale[n][1] = v2.y;
      }
      // 16 bytes of a row become 16 numbers of 16 bits: two chunks of the row's 256 bytes
#pragma unroll
      for (int e = 0; e < 2 * L::kTok * 8 / (32 * kWarps); ++e) {
        constexpr int kStep = 32 * kWarps;
        const int i = e * kStep + threadIdx.x, r = i >> 3, c = i & 7;         // rows 0-31 Keys, 32-63 Values
        const bool value = e * kStep >= L::kTok * 8;
        const uint4 w = *reinterpret_cast<const uint4 *>(raw + at<128>(r, c));
        const uint32_t in[4] = {w.x, w.y, w.z, w.w};
        uint32_t out[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint16_t two = (uint16_t)(in[k >> 1] >> (16 * (k & 1)));
          out[k] = value ? e4m3x2_bf16x2(two) : e4m3x2_16<T>(two);
        }
        *reinterpret_cast<uint4 *>(smem + L::kTile + at<256>(r, 2 * c)) = make_uint4(out[0], out[1], out[2], out[3]);
        *reinterpret_cast<uint4 *>(smem + L::kTile + at<256>(r, 2 * c + 1)) = make_uint4(out[4], out[5], out[6], out[7]);
      }
      __syncthreads();
      k_addr = smem_u32(smem + L::kTile);
      v_addr = k_addr + L::kTok * 256;
    } else {
      k_addr = smem_u32(raw);
      v_addr = k_addr + L::kTok * 256;
    }
    if (!busy) continue;
    if (all_see < min(t1, first + L::kTok)) {        // tokens that some rows do not see
      const int s0 = max(all_see - first, 0), s1 = min(t1 - first, L::kTok);
      unsigned char *v = smem + (FP8 ? L::kTile : L::kRing + tile % L::kStages * L::kRaw) + L::kTok * 256;
      if (any_not_finite<MV>(v, s0, s1)) {
        take_apart<MV>(v, s0, s1, first, apart_s);
        apart = true;
      }
      if constexpr (FP8) apart |= scales_apart(raw + L::kScales + 128, vscale, s0, s1, first, apart_s);
    }
    float s[kNT][4];
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.f;
    const uint32_t k_lane = k_addr + k_at, k_lane2 = k_lane + 16 * 256, v_lane = v_addr + v_at, v_lane2 = v_lane + 16 * 256;
#pragma unroll
    for (int k = 0; k < 8; ++k) {                    // 16 channels
      uint32_t qa[4], r[4], r2[4];
      ldmatrix_x4(even(q_lane, 2 * k), qa[0], qa[1], qa[2], qa[3]);
      ldmatrix_x4(even(k_lane, 2 * k), r[0], r[1], r[2], r[3]);
      ldmatrix_x4(even(k_lane2, 2 * k), r2[0], r2[1], r2[2], r2[3]);
      mma_16816<T>(s[0], qa, r[0], r[1]);
      mma_16816<T>(s[1], qa, r[2], r[3]);
      mma_16816<T>(s[2], qa, r2[0], r2[1]);
      mma_16816<T>(s[3], qa, r2[2], r2[3]);
    }
    if constexpr (FP8) {
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] *= kscale[n][i & 1];
    }
    if (first + L::kTok > all_see) {                 // unseen tokens weigh nothing
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (first + n * 8 + 2 * j4 + (i & 1) >= limit[i >> 1]) s[n][i] = -INFINITY;
    }
    bool grow[2];
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx[i >> 1] = fmaxf(mx[i >> 1], s[n][i]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2)) * a.scale_log2;
      grow[i] = mx[i] > m[i] + kLazy;
    }
    if (__any_sync(0xffffffffu, grow[0] || grow[1])) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float f = grow[i] ? fast_exp2(m[i] - mx[i]) : 1.f;
        if (grow[i]) m[i] = mx[i];
        l[i] *= f;
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          acc[n][2 * i] *= f;
          acc[n][2 * i + 1] *= f;
        }
      }
    }
    const float base[2] = {m[0] > -INFINITY ? m[0] : 0.f, m[1] > -INFINITY ? m[1] : 0.f};
    uint32_t pa[kNT][2], pl[kNT][2];                 // Phi, Plo
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float w0 = fast_exp2(fmaf(s[n][2 * i], a.scale_log2, -base[i])), w1 = fast_exp2(fmaf(s[n][2 * i + 1], a.scale_log2, -base[i]));
        l[i] += w0 + w1;
        if constexpr (FP8) {
          w0 *= vscale[n][0];
          w1 *= vscale[n][1];
        }
        two_parts<MV>(w0, w1, pa[n][i], pl[n][i]);
      }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {                 // 16 tokens
      const uint32_t pf[4] = {pa[2 * kk][0], pa[2 * kk][1], pa[2 * kk + 1][0], pa[2 * kk + 1][1]};
      const uint32_t pg[4] = {pl[2 * kk][0], pl[2 * kk][1], pl[2 * kk + 1][0], pl[2 * kk + 1][1]};
#pragma unroll
      for (int c = 0; c < 16; c += 2) {              // two chunks of 8 channels
        uint32_t r[4];
        ldmatrix_x4_trans(even(kk ? v_lane2 : v_lane, c), r[0], r[1], r[2], r[3]);
        mma_16816<MV>(acc[c], pf, r[0], r[1]);
        mma_16816<MV>(acc[c + 1], pf, r[2], r[3]);
        mma_16816<MV>(acc[c], pg, r[0], r[1]);
        mma_16816<MV>(acc[c + 1], pg, r[2], r[3]);
      }
    }
  }
  cp_async_wait_all();
  if (__syncthreads_or(apart)) {
#pragma unroll
    for (int n = 0; n < 16; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (limit[i >> 1] > apart_s[8 * n + 2 * j4 + (i & 1)]) acc[n][i] = NAN;
  }
  const long long slot = (long long)bh * p.chunks + chunk;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float ll = l[i];
    ll += __shfl_xor_sync(0xffffffffu, ll, 1);
    ll += __shfl_xor_sync(0xffffffffu, ll, 2);
    const int r = row0 + g + 8 * i;
    if (r < p.rows) {
      // channels 8 n + 2 j4, + 1: half of channel group 2 n + j4 / 2
      float *out = p.acc + ((slot * 32 + (j4 >> 1)) * p.rows + r) * 4 + 2 * (j4 & 1);
#pragma unroll
      for (int n = 0; n < 16; ++n)
        *reinterpret_cast<float2 *>(out + 8ll * n * p.rows) =
            make_float2(acc[n][2 * i], acc[n][2 * i + 1]);
      // NaN logits: m NaN too, as no weight may drop them
      if (j4 == 0) reinterpret_cast<float2 *>(p.ml)[slot * p.rows + r] = make_float2(isnan(ll) ? ll : m[i], ll);
    }
  }
  end_after_previous();
}

template <typename T, bool FP8>
cudaError_t launch_rows(const TextParams &p, cudaStream_t stream) {
  const int smem = RowsSmem<FP8>::kBytes;
  cudaError_t e = allow_shared_memory<shared_text_rows_kernel<T, FP8>>(smem);
  if (e != cudaSuccess) return e;
  const dim3 grid(p.s.prefixes * p.s.questions * p.s.kv_heads, p.chunks, (p.rows + 63) / 64);
  if (p.beside) return launch_overlapping(shared_text_rows_kernel<T, FP8>, grid, dim3(kWarps * 32), smem, stream, p);
  shared_text_rows_kernel<T, FP8><<<grid, kWarps * 32, smem, stream>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_few(const TextParams &p, cudaStream_t stream) {
  cudaError_t e = allow_shared_memory<shared_text_kernel<T>>(TextSmem::kBytes);
  if (e != cudaSuccess) return e;
  const dim3 grid(p.s.prefixes * p.s.questions * p.s.kv_heads, p.chunks);
  if (p.beside) return launch_overlapping(shared_text_kernel<T>, grid, dim3(kWarps * 32), TextSmem::kBytes, stream, p);
  shared_text_kernel<T><<<grid, kWarps * 32, TextSmem::kBytes, stream>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch(const TextParams &p, cudaStream_t stream) {
  if (!p.s.text_fp8) return launch_rows<T, false>(p, stream);
  return p.rows <= 16 ? launch_few<T>(p, stream) : launch_rows<T, true>(p, stream);
}

}  // namespace

cudaError_t launch_shared_text(const TextParams &p, cudaStream_t stream) {
  return p.s.dtype == 1 ? launch<__nv_bfloat16>(p, stream) : launch<__half>(p, stream);
}

}  // namespace rtk
