// Shared-prefix attention, the prefix part, on the 5th-generation tensor cores.
//
// The queries of all N questions, T tokens and G heads of a (prefix, KV head) are
// rows of one matrix: up to 128 of them meet every prefix token in one
// tcgen05.mma, so a prefix's Keys and Values come from HBM once however many
// questions share it.  Per unit of 128 rows (shared.h: PrefixSplit) and per
// block of tokens:
//
//   S  = Q . K^T        prompt block, 64 tokens, K = 128 channels
//   S  = [Qhi | Qlo] . [K~ | K~]^T    visual block, 128 tokens, K = 2 D_keep: the rotated
//                       query q~ = q R is taken in fp32 and split into two 16-bit parts
//                       (one part alone would move logits by 2^-9)
//   x  = c (S + q . delta_mu),  c = log2(e) / sqrt(D)     (delta_mu: visual blocks)
//   P  = 2^(x - m) rounded to 16 bits, the MMA's operand type; l sums it unrounded
//   O += P . V
//
// m follows the running maximum lazily: O and l are rescaled only when a maximum
// grows by more than 2^8 over the one in use (P stays below 2^8, O and l are fp32).
//
// CTA (one per SM, 12 warps):
//   warp 0      TMA producer: a ring of stages, one block's K and V each
//   warp 1      TMEM owner; one lane issues the MMAs
//   warps 4-7   softmax of the even blocks: thread = query row (TMEM lane)
//   warps 8-11  softmax of the odd blocks
// Even and odd blocks are two independent streams, each with its own S / P columns,
// (m, l) and O accumulator in TMEM (2 x 128 + 2 x 128 = all 512 columns): while one
// stream's softmax runs, the tensor core works for the other.  P goes back over S
// (its upper half) in TMEM as the A operand of P . V.  At the end of a unit the streams are joined and
// the partial result of (unit, CTA) is written for shared_merge.cu.
#include <type_traits>

#include "shared.h"
#include "tcgen05.cuh"

namespace rtk {
namespace {

constexpr int kThreads = 384;
constexpr int kFullTok = 64, kVisTok = 128;
constexpr uint32_t kColsS = 128;                 // TMEM columns of a stream's S / P
constexpr uint32_t kColP = 64;                   // P within them: over the upper half of S
constexpr uint32_t kColO = 2 * kColsS;           // first column of the O accumulators
constexpr float kLazy = 8.f;

template <int DK>
struct PrefixSmem {
  static constexpr int kKeyBytes = kVisTok * DK * 2;
  static constexpr int kStage = kKeyBytes + kVisTok * 256;         // a visual block (a prompt block is 32 KB)
  static_assert(kStage >= kFullTok * 512 && kStage % 1024 == 0, "stage");
  static constexpr int kStages = DK == 64 ? 3 : 4;
  static constexpr int kQ = 0;                                     // Q: 2 boxes of 128 rows x 64 channels
  static constexpr int kRot = kQ + 32768;                          // [Qhi | Qlo]; before it R^T
  static constexpr int kRotBytes = DK == 64 ? 32768 : 16384;
  static constexpr int kRing = kRot + kRotBytes;
  static constexpr int kBias = kRing + kStages * kStage;           // float[128]
  static constexpr int kDm = kBias + 512;                          // float[128]
  static constexpr int kMl = kDm + 512;                            // float2[2][128]
  static constexpr int kBar = kMl + 2048;
  // full[S], empty[S], s_ready[2], p_ready[2], rot, o_done
  static constexpr int kNumBars = 2 * kStages + 6;
  static constexpr int kTmemSlot = kBar + kNumBars * 8;
  static constexpr int kAbort = kTmemSlot + 4;
  static constexpr int kBytes = kAbort + 4;
  static_assert(kBytes + 1024 <= 232448, "shared memory budget");
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

struct RowStat {
  float m, l;
};

// O of this warp's rows times each row's f.
__device__ __forceinline__ void rescale_o(uint32_t o, float f) {
#pragma unroll 1
  for (int c = 0; c < 128; c += 16) {
    uint32_t r[16];
    tmem_ld16_nowait(o + c, r);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f);
    tmem_st16_nowait(o + c, r);
  }
}

// 64 columns of S; those that do not count become -inf, whatever was there.
__device__ __forceinline__ void load_half(uint32_t s, bool all, uint32_t v0, uint32_t v1, uint32_t (&r)[2][32]) {
  tmem_ld32_nowait(s, r[0]);
  tmem_ld32_nowait(s + 32, r[1]);
  tmem_wait_ld();
  if (!all) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (!((v0 >> i) & 1u)) r[0][i] = 0xff800000u;
      if (!((v1 >> i) & 1u)) r[1][i] = 0xff800000u;
    }
  }
}

__device__ __forceinline__ float max_half(const uint32_t (&r)[2][32]) {
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int i = 0; i < 32; i += 2)
      mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(r[c][i]), __uint_as_float(r[c][i + 1]));
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}

// Weights of 64 columns: 32 columns of P (16-bit pairs) at `p`, their sum into l.
template <typename T>
__device__ __forceinline__ void weights_half(uint32_t p, const uint32_t (&r)[2][32], float2 scale, float2 off,
                                             float2 (&l)[2]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float2 x = __ffma2_rn(make_float2(__uint_as_float(r[c][2 * i]), __uint_as_float(r[c][2 * i + 1])), scale, off);
      x.x = fast_exp2(x.x);
      x.y = fast_exp2(x.y);
      l[i & 1] = __fadd2_rn(l[i & 1], x);
      w[i] = pack2<T>(x.x, x.y);
    }
    tmem_st16_nowait(p + 16 * c, w);
  }
}

// One block of one stream for this thread's row: S in TMEM columns [s, s + 64 or 128),
// P written to [s + 64, s + 128), m / l / O brought along.  `valid` (a bit per token) marks the
// tokens that count; `all` = every one does.  64 columns are in registers at a time;
// of a visual block the upper half stays there from the maximum to the weights (P
// goes over it) and the lower half is read again.
template <typename T, bool VIS>
__device__ __forceinline__ void softmax_block(uint32_t s, uint32_t o, bool first, float scale, float bias, bool all,
                                              const uint32_t (&valid)[4], RowStat &st) {
  uint32_t r[2][32];
  load_half(s, all, valid[0], valid[1], r);
  float mx = max_half(r);
  if constexpr (VIS) {
    load_half(s + 64, all, valid[2], valid[3], r);
    mx = fmaxf(mx, max_half(r));
  }
  const float top = fmaf(mx, scale, bias);           // scale > 0; -inf stays -inf
  const bool grow = top > st.m + kLazy;              // from -inf: whenever there is a maximum
  if (__any_sync(0xffffffffu, grow)) {
    const float m2 = grow ? top : st.m;
    const float f = grow ? fast_exp2(st.m - m2) : 1.f;      // first maximum: 2^-inf = 0
    st.m = m2;
    st.l *= f;
    if (!first) rescale_o(o, f);
  }
  const float off = bias - (st.m > -INFINITY ? st.m : 0.f);
  const float2 scale2 = make_float2(scale, scale), off2 = make_float2(off, off);
  float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  if constexpr (VIS) {
    weights_half<T>(s + kColP + 32, r, scale2, off2, l2);
    load_half(s, all, valid[0], valid[1], r);
  }
  weights_half<T>(s + kColP, r, scale2, off2, l2);
  st.l += (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
  tmem_wait_st();
}

template <typename T, int DK>
__global__ void __launch_bounds__(kThreads, 1)
    shared_prefix_kernel(const __grid_constant__ PrefixMaps maps, const __grid_constant__ PrefixParams p) {
  using L = PrefixSmem<DK>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char *smem = reinterpret_cast<unsigned char *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t *full_bar = reinterpret_cast<uint64_t *>(smem + L::kBar);
  uint64_t *empty_bar = full_bar + L::kStages;
  uint64_t *s_bar = empty_bar + L::kStages;       // [2] S of the stream's block is in TMEM
  uint64_t *p_bar = s_bar + 2;                    // [2] P of the stream's block is in TMEM
  uint64_t *rot_bar = p_bar + 2;                  // rotated queries are in TMEM
  uint64_t *o_bar = rot_bar + 1;                  // both O accumulators are complete
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::kTmemSlot);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::kAbort);
  float *bias_s = reinterpret_cast<float *>(smem + L::kBias);
  float *dm_s = reinterpret_cast<float *>(smem + L::kDm);
  float2 *ml_s = reinterpret_cast<float2 *>(smem + L::kMl);

  const PrefixSplit &sp = p.split;
  const SharedParams &a = p.s;
  const int cta = blockIdx.x;
  const long long r0 = sp.range_begin(cta), r1 = sp.range_begin(cta + 1);
  const int u0 = (int)(r0 / sp.unit_weight), u1 = (int)((r1 - 1) / sp.unit_weight);   // r1 > r0
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_bar[i], 1);
      mbar_init(&p_bar[i], 4);
    }
    mbar_init(rot_bar, 1);
    mbar_init(o_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ---------------------------------------------------------------- producer
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int u = u0; u <= u1 && ok; ++u) {
        const long long w = (long long)u * sp.unit_weight;
        const int j0 = r0 > w ? sp.block_from((int)(r0 - w)) : 0;
        const int j1 = r1 - w >= sp.unit_weight ? sp.blocks() : sp.block_from((int)(r1 - w));
        const int ph = u / sp.row_tiles, pre = ph / a.kv_heads, h = ph % a.kv_heads;
        for (int j = j0; j < j1; ++j, ++it) {
          const int stg = it % L::kStages;
          if (!mbar_wait_bounded(&empty_bar[stg], ((it / L::kStages) & 1) ^ 1, abort_flag, p.status)) {
            ok = false;
            break;
          }
          unsigned char *dst = smem + L::kRing + stg * L::kStage;
          if (j < sp.blocks_full) {
            mbar_arrive_expect_tx(&full_bar[stg], kFullTok * 512);
            tma_load_4d(dst, &maps.kf, 0, j * kFullTok, h, pre, &full_bar[stg]);
            tma_load_4d(dst + 8192, &maps.kf, 64, j * kFullTok, h, pre, &full_bar[stg]);
            tma_load_4d(dst + 16384, &maps.vf, 0, j * kFullTok, h, pre, &full_bar[stg]);
            tma_load_4d(dst + 24576, &maps.vf, 64, j * kFullTok, h, pre, &full_bar[stg]);
          } else {
            const int tok = (j - sp.blocks_full) * kVisTok;
            mbar_arrive_expect_tx(&full_bar[stg], L::kStage);
            tma_load_4d(dst, &maps.ks, 0, tok, h, pre, &full_bar[stg]);
            tma_load_4d(dst + L::kKeyBytes, &maps.vs, 0, tok, h, pre, &full_bar[stg]);
            tma_load_4d(dst + L::kKeyBytes + 16384, &maps.vs, 64, tok, h, pre, &full_bar[stg]);
          }
        }
      }
      if (*abort_flag) {                     // let the copies in flight land before the CTA exits
        int dead = 0;
        for (int k = it > L::kStages ? it - L::kStages : 0; k < it; ++k)
          mbar_wait_bounded(&full_bar[k % L::kStages], (k / L::kStages) & 1, &dead, p.status);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    constexpr uint32_t kFmt = kBf16 ? 1u : 0u;
    constexpr uint32_t kIdRot = idesc_f16(kFmt, 0, 0, 128, DK);
    constexpr uint32_t kIdFull = idesc_f16(kFmt, 0, 0, 128, kFullTok);
    constexpr uint32_t kIdVis = idesc_f16(kFmt, 0, 0, 128, kVisTok);
    constexpr uint32_t kIdPv = idesc_f16(kFmt, 0, 1, 128, 128);
    const uint32_t q_addr = smem_u32(smem + L::kQ), rot_addr = smem_u32(smem + L::kRot);
    int it = 0;
    uint32_t np = 0;                         // parities of the next P block, a bit per stream
    for (int u = u0; u <= u1; ++u) {
      const long long w = (long long)u * sp.unit_weight;
      const int j0 = r0 > w ? sp.block_from((int)(r0 - w)) : 0;
      const int j1 = r1 - w >= sp.unit_weight ? sp.blocks() : sp.block_from((int)(r1 - w));
      if (j0 >= j1) continue;
      named_barrier_sync(1, 288);            // Q and R^T are in shared memory
      if (j1 > sp.blocks_full) {
        if (lane == 0) {
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_f16(tmem, smem_desc_kmajor<128>(q_addr + (k >> 2) * 16384 + (k & 3) * 32),
                     smem_desc_kmajor<128>(rot_addr + (k >> 2) * (DK * 128) + (k & 3) * 32), kIdRot, k > 0);
          umma_commit(rot_bar);
        }
        __syncwarp();
        named_barrier_sync(1, 288);          // [Qhi | Qlo] is in shared memory
      }
      if (lane == 0) {
        tc_fence_after();
        auto issue_qk = [&](int j, int i) {
          const int stg = i % L::kStages, x = (j - j0) & 1;
          mbar_wait_bounded(&full_bar[stg], (i / L::kStages) & 1, abort_flag, p.status);
          tc_fence_after();
          const uint32_t k_addr = smem_u32(smem + L::kRing + stg * L::kStage);
          const uint32_t d = tmem + x * kColsS;
          if (j < sp.blocks_full) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              umma_f16(d, smem_desc_kmajor<128>(q_addr + (k >> 2) * 16384 + (k & 3) * 32),
                       smem_desc_kmajor<128>(k_addr + (k >> 2) * 8192 + (k & 3) * 32), kIdFull, k > 0);
          } else {
            constexpr int kSteps = DK / 16;
#pragma unroll
            for (int k = 0; k < 2 * kSteps; ++k) {
              const int col = 16 * k;        // of [Qhi | Qlo]
              umma_f16(d, smem_desc_kmajor<128>(rot_addr + (col >> 6) * 16384 + (col & 63) * 2),
                       smem_desc_kmajor<DK * 2>(k_addr + (k % kSteps) * 32), kIdVis, k > 0);
            }
          }
          umma_commit(&s_bar[x]);
        };
        issue_qk(j0, it);
        if (j0 + 1 < j1) issue_qk(j0 + 1, it + 1);
        for (int j = j0; j < j1; ++j, ++it) {
          const int x = (j - j0) & 1, stg = it % L::kStages;
          mbar_wait_bounded(&p_bar[x], (np >> x) & 1, abort_flag, p.status);
          np ^= 1u << x;
          tc_fence_after();
          const bool vis = j >= sp.blocks_full;
          const uint32_t v_addr = smem_u32(smem + L::kRing + stg * L::kStage) + (vis ? L::kKeyBytes : 16384);
          const uint32_t d = tmem + kColO + x * 128, pa = tmem + x * kColsS + kColP;
          const uint32_t half = vis ? 16384u : 8192u;
          const int steps = vis ? kVisTok / 16 : kFullTok / 16;
          for (int k = 0; k < steps; ++k)
            umma_f16_ts(d, pa + 8 * k, smem_desc_sw128(v_addr + k * 2048, half, 1024), kIdPv, k > 0 || j - j0 > 1);
          umma_commit(&empty_bar[stg]);
          if (j + 1 == j1) umma_commit(o_bar);
          if (j + 2 < j1) issue_qk(j + 2, it + 2);
        }
      }
      __syncwarp();
      named_barrier_sync(1, 288);            // the unit's partial has been read out
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- softmax
    const int x = (warp - 4) >> 2;                   // stream
    const int tid = threadIdx.x - 128;               // 0 .. 255
    const int row = tid & 127;                       // query row of the unit = TMEM lane
    const uint32_t lanes = (uint32_t)(row & ~31) << 16;
    const uint32_t s_col = tmem + lanes + x * kColsS, o_col = tmem + lanes + kColO + x * 128;
    uint32_t ns = 0, nrot = 0, no = 0;
    for (int u = u0; u <= u1; ++u) {
      const long long w = (long long)u * sp.unit_weight;
      const int j0 = r0 > w ? sp.block_from((int)(r0 - w)) : 0;
      const int j1 = r1 - w >= sp.unit_weight ? sp.blocks() : sp.block_from((int)(r1 - w));
      if (j0 >= j1) continue;
      const int ph = u / sp.row_tiles, pre = ph / a.kv_heads, h = ph % a.kv_heads;
      const int base = (u % sp.row_tiles) * 128;
      const int live = min(128, sp.rows - base);     // rows of this unit
      const bool vis = j1 > sp.blocks_full;
      {
        // queries: thread = half a row (8 chunks of 16 bytes)
        const int qrow = tid >> 1, half = tid & 1;
        const bool there = qrow < live;
        const T *src = nullptr;
        if (there) {
          const int r = base + qrow, g = r % a.groups, nt = r / a.groups;
          src = static_cast<const T *>(a.q.data) + ((long long)pre * a.questions + nt / a.tokens) * a.q.s[0] +
                (nt % a.tokens) * a.q.s[1] + (h * a.groups + g) * a.q.s[2] + half * 64;
        }
        unsigned char *dst = smem + L::kQ + half * 16384;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const uint4 v = there ? __ldg(reinterpret_cast<const uint4 *>(src) + c) : make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4 *>(dst + swizzled_offset<128>(qrow, c * 8)) = v;
        }
        if (vis) {
          // R^T, K-major: row j holds column j of R
          const T *R = static_cast<const T *>(a.R.data) + pre * a.R.s[0] + h * a.R.s[1];
          const uint32_t rt = smem_u32(smem + L::kRot);
          if (p.R_rows) {                              // rows of R in 16-byte pieces
            for (int e = tid; e < 128 * DK / 8; e += 256) {
              const int d = e / (DK / 8), c = e % (DK / 8);
              const uint4 v = __ldg(reinterpret_cast<const uint4 *>(R + d * a.R.s[2] + c * 8));
              const uint32_t words[4] = {v.x, v.y, v.z, v.w};
              const uint32_t box = rt + (d >> 6) * (DK * 128);
#pragma unroll
              for (int i = 0; i < 8; ++i)
                st_shared_u16(box + swizzled_offset<128>(c * 8 + i, (d & 63) & ~7) + (d & 7) * 2,
                              (uint16_t)(words[i >> 1] >> (16 * (i & 1))));
            }
          } else {                                     // any strides; a transposed R reads along its columns
#pragma unroll 8
            for (int e = tid; e < 128 * DK; e += 256) {
              const int d = e & 127, j = e >> 7;
              st_shared_u16(rt + (d >> 6) * (DK * 128) + swizzled_offset<128>(j, (d & 63) & ~7) + (d & 7) * 2,
                            __ldg(reinterpret_cast<const unsigned short *>(R + d * a.R.s[2] + j * a.R.s[3])));
            }
          }
          if (tid < 128)
            dm_s[tid] = a.dm.data != nullptr
                            ? to_f32(static_cast<const T *>(a.dm.data)[pre * a.dm.s[0] + h * a.dm.s[1] + tid])
                            : 0.f;
        }
      }
      fence_proxy_async_smem();
      named_barrier_sync(1, 288);
      if (vis) {
        if (x == 0) {
          // rotated queries out of TMEM, as two 16-bit parts into shared memory
          mbar_wait_bounded(rot_bar, nrot & 1, abort_flag, p.status);
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < DK; c += 16) {
            uint32_t r[16];
            tmem_ld16_nowait(tmem + lanes + c, r);
            tmem_wait_ld();
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float f0 = __uint_as_float(r[2 * i]), f1 = __uint_as_float(r[2 * i + 1]);
              hi[i] = pack2<T>(f0, f1);
              float h0, h1;
              unpack2<T>(hi[i], h0, h1);
              lo[i] = pack2<T>(f0 - h0, f1 - h1);
            }
            const uint32_t rot = smem_u32(smem + L::kRot);
            const int cl = DK + c;             // column of the low parts
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              st_shared_v4(rot + (c >> 6) * 16384 + swizzled_offset<128>(row, (c & 63) + 8 * i), hi[4 * i],
                           hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]);
              st_shared_v4(rot + (cl >> 6) * 16384 + swizzled_offset<128>(row, (cl & 63) + 8 * i), lo[4 * i],
                           lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
            }
          }
          tc_fence_before();
        } else {
          float b = 0.f;
          if (a.dm.data != nullptr) {
            const unsigned char *q = smem + L::kQ;
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const uint4 v = *reinterpret_cast<const uint4 *>(q + (c >> 3) * 16384 + swizzled_offset<128>(row, (c & 7) * 8));
              const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float lo, hi;
                unpack2<T>(words[i], lo, hi);
                b = fmaf(lo, dm_s[c * 8 + 2 * i], b);
                b = fmaf(hi, dm_s[c * 8 + 2 * i + 1], b);
              }
            }
          }
          bias_s[row] = b * a.scale_log2;
        }
        ++nrot;
        fence_proxy_async_smem();
        named_barrier_sync(1, 288);
      }
      const float bias = vis ? bias_s[row] : 0.f;
      RowStat st{-INFINITY, 0.f};
      const bool busy = (row & ~31) < live;          // some row of this warp exists
      for (int j = j0 + x; j < j1; j += 2, ++ns) {
        uint32_t valid[4] = {~0u, ~0u, ~0u, ~0u};
        bool all = true;
        const bool full = j < sp.blocks_full;
        if (full) {
          const int tok = j * kFullTok, left = a.seq_full - tok;
          if (a.mask.data != nullptr || left < kFullTok) {
            const uint8_t *mk = static_cast<const uint8_t *>(a.mask.data) + pre * a.mask.s[0];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int t = 32 * i + lane;
              const bool in = t < left && (a.mask.data == nullptr || mk[(tok + t) * a.mask.s[1]] != 0);
              valid[i] = __ballot_sync(0xffffffffu, in);
            }
            all = (valid[0] & valid[1]) == ~0u;
          }
        } else {
          const int left = a.seq_sparse - (j - sp.blocks_full) * kVisTok;
          if (left < kVisTok) {
            all = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int n = left - 32 * i;
              valid[i] = n >= 32 ? ~0u : n > 0 ? (1u << n) - 1u : 0u;
            }
          }
        }
        mbar_wait_bounded(&s_bar[x], ns & 1, abort_flag, p.status);
        tc_fence_after();
        if (full && !all && a.mask.data != nullptr) {
          // a masked token's Values may hold anything, and 0 * NaN is NaN: zero them
          unsigned char *v = smem + L::kRing;
          // the stage of this block: blocks are numbered along the CTA's whole range
          long long before = 0;
          for (int q = u0; q < u; ++q) {
            const long long wq = (long long)q * sp.unit_weight;
            const int b0 = r0 > wq ? sp.block_from((int)(r0 - wq)) : 0;
            before += sp.blocks() - b0;
          }
          v += ((before + (j - j0)) % L::kStages) * L::kStage + 16384;
          for (int t = (warp & 3); t < kFullTok; t += 4)
            if (!(((t < 32 ? valid[0] : valid[1]) >> (t & 31)) & 1u))
              *reinterpret_cast<uint2 *>(v + (lane >> 4) * 8192 + t * 128 + (lane & 15) * 8) = make_uint2(0, 0);
          fence_proxy_async_smem();
        }
        if (busy) {
          if (full)
            softmax_block<T, false>(s_col, o_col, j - j0 < 2, a.scale_log2, 0.f, all, valid, st);
          else
            softmax_block<T, true>(s_col, o_col, j - j0 < 2, a.scale_log2, bias, all, valid, st);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_bar[x]);
      }
      // join the two streams: each warp group writes 64 channels of the row
      ml_s[x * 128 + row] = make_float2(st.m, st.l);
      mbar_wait_bounded(o_bar, no & 1, abort_flag, p.status);
      ++no;
      tc_fence_after();
      named_barrier_sync(2, 256);
      const float2 e0 = ml_s[row], e1 = ml_s[128 + row];
      const float m = fmaxf(e0.x, e1.x);
      const float f0 = e0.x > -INFINITY ? fast_exp2(e0.x - m) : 0.f;
      const float f1 = e1.x > -INFINITY ? fast_exp2(e1.x - m) : 0.f;
      const bool two = j1 - j0 > 1;                  // the odd stream had a block
      const long long slot = u + cta;
      if (busy) {
        float *out = p.acc + (slot * 128 + row) * 128 + 64 * x;
        const uint32_t c0 = tmem + lanes + kColO + 64 * x, c1 = c0 + 128;
#pragma unroll
        for (int c = 0; c < 64; c += 16) {
          uint32_t ra[16], rb[16];
          tmem_ld16_nowait(c0 + c, ra);
          if (two) tmem_ld16_nowait(c1 + c, rb);
          tmem_wait_ld();
          if (row < live) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              float v[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                v[k] = f0 > 0.f ? __uint_as_float(ra[i + k]) * f0 : 0.f;
                if (two && f1 > 0.f) v[k] = fmaf(__uint_as_float(rb[i + k]), f1, v[k]);
              }
              *reinterpret_cast<float4 *>(out + c + i) = make_float4(v[0], v[1], v[2], v[3]);
            }
          }
        }
        if (x == 0 && row < live)
          reinterpret_cast<float2 *>(p.ml)[slot * 128 + row] = make_float2(m, e0.y * f0 + e1.y * f1);
      }
      tc_fence_before();
      named_barrier_sync(1, 288);
    }
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int DK>
cudaError_t launch(const PrefixMaps &maps, const PrefixParams &p, cudaStream_t stream) {
  const int smem = PrefixSmem<DK>::kBytes + 1024;
  cudaError_t e = cudaFuncSetAttribute(shared_prefix_kernel<T, DK>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  shared_prefix_kernel<T, DK><<<p.split.grid, kThreads, smem, stream>>>(maps, p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_shared_prefix(const PrefixMaps &maps, const PrefixParams &p, cudaStream_t stream) {
  const bool bf = p.s.dtype == 1;
  switch (p.s.head_dim_keep) {
    case 16: return bf ? launch<__nv_bfloat16, 16>(maps, p, stream) : launch<__half, 16>(maps, p, stream);
    case 32: return bf ? launch<__nv_bfloat16, 32>(maps, p, stream) : launch<__half, 32>(maps, p, stream);
    case 64: return bf ? launch<__nv_bfloat16, 64>(maps, p, stream) : launch<__half, 64>(maps, p, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace rtk
