// Shared-prefix attention, the prefix part, on the 5th-generation tensor cores.
//
// The queries of all N questions, T tokens and G heads of a (prefix, KV head) are
// rows of one matrix: up to 128 of them meet every prefix token in one
// tcgen05.mma, so a prefix's Keys and Values come from HBM once however many
// questions share it.  Per unit of 128 rows (shared.h: PrefixSplit) and per
// block of tokens:
//
//   S  = Q . K^T        prompt block, 64 tokens, K = 128 channels
//   S  = [Qhi | Qlo] . [K~ | K~]^T    visual block, 128 tokens (two sub-blocks), K = 2 D_keep: the rotated
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
//   warps 1, 2  issue the MMAs of the even and the odd sub-blocks (one elected lane each:
//               a single thread's instructions could not keep the tensor core fed); warp 1
//               owns the TMEM
//   warps 4-7   softmax of the even sub-blocks: thread = query row (TMEM lane)
//   warps 8-11  softmax of the odd sub-blocks
// A sub-block is 64 tokens: a prompt block, or half a visual block.  Even and odd
// sub-blocks are two independent streams with their own (m, l) and O accumulator in
// TMEM (2 x 128 columns), and two S buffers each (2 x 2 x 64 columns: all 512): while
// a warp group works on one, the tensor core turns the other into the next S.  P goes
// over S in TMEM as the A operand of P . V.  At the end of a unit the streams are
// joined and the partial result of (unit, CTA) is written for shared_merge.cu.
#include <type_traits>

#include "shared.h"
#include "tcgen05.cuh"

namespace rtk {
namespace {

constexpr int kThreads = 384;
constexpr int kFullTok = 64, kVisTok = 128;      // tokens of a block
constexpr int kSub = 64;                         // tokens of a sub-block
constexpr uint32_t kColsS = 64;                  // TMEM columns of an S buffer
constexpr uint32_t kColO = 4 * kColsS;           // first column of the O accumulators
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
  // full[S], empty[S], s_ready[4], p_ready[4], pv[2], rot, o_done
  static constexpr int kNumBars = 2 * kStages + 12;
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

// One sub-block for this thread's row: S in TMEM columns [s, s + 64), P written to
// [s, s + 32), m and l brought along; rescale(f) multiplies O by each row's f when the
// reference of any row of the warp moves; before() comes before the exponentials.  v0, v1 (a bit per token) mark the tokens that
// count; `all` = every one does.
template <typename T, typename Rescale, typename Before>
__device__ __forceinline__ void softmax_sub(uint32_t s, float scale, float bias, bool all, uint32_t v0, uint32_t v1,
                                            RowStat &st, Rescale rescale, Before before) {
  uint32_t r[2][32];
  tmem_ld32_nowait(s, r[0]);
  tmem_ld32_nowait(s + 32, r[1]);
  tmem_wait_ld();
  if (!all) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {                   // -inf, whatever was there
      if (!((v0 >> i) & 1u)) r[0][i] = 0xff800000u;
      if (!((v1 >> i) & 1u)) r[1][i] = 0xff800000u;
    }
  }
  float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int i = 0; i < 32; i += 2)
      mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(r[c][i]), __uint_as_float(r[c][i + 1]));
  // scale > 0; -inf stays -inf
  const float top = fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), scale, bias);
  const bool grow = top > st.m + kLazy;              // from -inf: whenever there is a maximum
  if (__any_sync(0xffffffffu, grow)) {
    const float m2 = grow ? top : st.m;
    const float f = grow ? fast_exp2(st.m - m2) : 1.f;      // first maximum: 2^-inf = 0
    st.m = m2;
    st.l *= f;
    rescale(f);
  }
  before();
  const float off = bias - (st.m > -INFINITY ? st.m : 0.f);
  const float2 scale2 = make_float2(scale, scale), off2 = make_float2(off, off);
  float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float2 x = __ffma2_rn(make_float2(__uint_as_float(r[c][2 * i]), __uint_as_float(r[c][2 * i + 1])), scale2, off2);
      x.x = fast_exp2(x.x);
      x.y = fast_exp2(x.y);
      l2[i & 1] = __fadd2_rn(l2[i & 1], x);
      w[i] = pack2<T>(x.x, x.y);
    }
    tmem_st16_nowait(s + 16 * c, w);
  }
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
  uint64_t *s_bar = empty_bar + L::kStages;       // [stream + 2 buffer] S is in TMEM
  uint64_t *p_bar = s_bar + 4;                    // [stream + 2 buffer] P is in TMEM
  uint64_t *pv_bar = p_bar + 4;                   // [stream] the P . V before the stream's last is done
  uint64_t *rot_bar = pv_bar + 2;                 // rotated queries are in TMEM
  uint64_t *o_bar = rot_bar + 1;                  // both O accumulators are complete
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::kTmemSlot);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::kAbort);
  float *bias_s = reinterpret_cast<float *>(smem + L::kBias);
  float *dm_s = reinterpret_cast<float *>(smem + L::kDm);
  float2 *ml_s = reinterpret_cast<float2 *>(smem + L::kMl);

  launch_dependents();
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
      mbar_init(&empty_bar[i], 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_bar[i], 1);
      mbar_init(&p_bar[i], 4);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&pv_bar[i], 1);
    mbar_init(rot_bar, 1);
    mbar_init(o_bar, 2);
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
  } else if (warp <= 2) {
    // ---------------------------------------------------------------- MMA issuers, one per stream
    const uint32_t x = warp - 1;
    constexpr uint32_t kFmt = kBf16 ? 1u : 0u;
    constexpr uint32_t kIdRot = idesc_f16(kFmt, 0, 0, 128, DK);
    constexpr uint32_t kIdQk = idesc_f16(kFmt, 0, 0, 128, kSub);
    constexpr uint32_t kIdPv = idesc_f16(kFmt, 0, 1, 128, 128);
    constexpr uint32_t kStep = L::kStage >> 4;       // from stage to stage, in a descriptor
    const uint32_t rot_addr = smem_u32(smem + L::kRot), ring = smem_u32(smem + L::kRing);
    const uint64_t q_desc = smem_desc_kmajor<128>(smem_u32(smem + L::kQ)), rot_desc = smem_desc_kmajor<128>(rot_addr);
    const uint64_t k_prompt = smem_desc_kmajor<128>(ring), v_prompt = smem_desc_sw128(ring + 16384, 8192, 1024);
    const uint32_t d_o = tmem + kColO + x * 128;
    int it = 0;                              // blocks of the segments before
    uint32_t np = 0;                         // parity of the next P of each buffer
    for (int u = u0; u <= u1; ++u) {
      const long long w = (long long)u * sp.unit_weight;
      const int j0 = r0 > w ? sp.block_from((int)(r0 - w)) : 0;
      const int j1 = r1 - w >= sp.unit_weight ? sp.blocks() : sp.block_from((int)(r1 - w));
      if (j0 >= j1) continue;
      named_barrier_sync(1, 320);            // Q and R^T are in shared memory
      if (j1 > sp.blocks_full) {
        if (x == 0 && elect_one()) {
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_f16_ss(tmem, q_desc + (((k >> 2) * 16384 + (k & 3) * 32) >> 4),
                        smem_desc_kmajor<128>(rot_addr + (k >> 2) * (DK * 128) + (k & 3) * 32), kIdRot, k > 0);
          umma_commit(rot_bar);
        }
        __syncwarp();
        named_barrier_sync(1, 320);          // [Qhi | Qlo] is in shared memory
      }
      if (elect_one()) {
        tc_fence_after();
        // Sub-block i of the segment: prompt blocks are one, visual blocks two; this
        // stream takes every other one, i = x, x + 2, ...: whole prompt blocks, and always
        // the same half of a visual block.  S runs two of them ahead of P . V: an S
        // buffer is free once the P . V that reads it is issued (the tensor core works
        // in order).  This thread's own instructions are what the tensor core waits for, so
        // stages and parities are carried along instead of being computed.
        const int nf = j0 < sp.blocks_full ? min(j1, sp.blocks_full) - j0 : 0;
        const int subs = nf + 2 * (j1 - j0 - nf);
        const uint32_t half = (x ^ (uint32_t)nf) & 1u;
        const uint64_t k_vis = smem_desc_kmajor<DK * 2>(ring + half * (kSub * DK * 2));
        const uint64_t v_vis = smem_desc_sw128(ring + L::kKeyBytes + half * 8192, 16384, 1024);
        uint32_t q_stage = (it + (x == 1 && nf > 0)) % L::kStages;
        uint32_t q_par = ((it + (x == 1 && nf > 0)) / L::kStages) & 1;
        uint32_t p_stage = q_stage;
        it += j1 - j0;
        auto issue_qk = [&](int i, uint32_t buf) {
          mbar_wait_bounded(&full_bar[q_stage], q_par, abort_flag, p.status);
          tc_fence_after();
          const uint32_t d = tmem + x * kColsS + buf * (2 * kColsS);
          if (i >= nf) {
            constexpr int kSteps = DK / 16;
            const uint64_t kd = k_vis + q_stage * kStep;
#pragma unroll
            for (int k = 0; k < 2 * kSteps; ++k) {
              const int col = 16 * k;        // of [Qhi | Qlo]
              umma_f16_ss(d, rot_desc + (((col >> 6) * 16384 + (col & 63) * 2) >> 4), kd + (((k % kSteps) * 32) >> 4),
                          kIdQk, k > 0);
            }
          } else {
            const uint64_t kd = k_prompt + q_stage * kStep;
#pragma unroll
            for (int k = 0; k < 8; ++k)
              umma_f16_ss(d, q_desc + (((k >> 2) * 16384 + (k & 3) * 32) >> 4),
                          kd + (((k >> 2) * 8192 + (k & 3) * 32) >> 4), kIdQk, k > 0);
          }
          umma_commit(&s_bar[x + 2 * buf]);
          q_stage += i + 2 <= nf ? 2 : 1;
          if (q_stage >= (uint32_t)L::kStages) {
            q_stage -= L::kStages;
            q_par ^= 1u;
          }
        };
        int i = x;
        if (i < subs) issue_qk(i, 0);
        if (i + 2 < subs) issue_qk(i + 2, 1);
        for (uint32_t buf = 0; i < subs; i += 2, buf ^= 1u) {
          mbar_wait_bounded(&p_bar[x + 2 * buf], (np >> buf) & 1u, abort_flag, p.status);
          np ^= 1u << buf;
          tc_fence_after();
          const uint32_t pa = tmem + x * kColsS + buf * (2 * kColsS);
          const uint64_t vd = (i >= nf ? v_vis : v_prompt) + p_stage * kStep;
#pragma unroll
          for (int k = 0; k < kSub / 16; ++k)
            umma_f16_ts(d_o, pa + 8 * k, vd + ((k * 2048) >> 4), kIdPv, k > 0 || i > 1);
          umma_commit(&empty_bar[p_stage]);            // two arrivals free a stage: one of each stream, or
          if (i < nf) umma_commit(&empty_bar[p_stage]);    // both of the one that has the prompt block
          p_stage += i + 2 <= nf ? 2 : 1;
          if (p_stage >= (uint32_t)L::kStages) p_stage -= L::kStages;
          if (i + 4 < subs) issue_qk(i + 4, buf);
          else if (i + 2 < subs) umma_commit(&pv_bar[x]);  // the P . V before the stream's last
        }
        umma_commit(o_bar);
      }
      __syncwarp();
      named_barrier_sync(1, 320);            // the unit's partial has been read out
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- softmax
    const int x = (warp - 4) >> 2;                   // stream
    const int tid = threadIdx.x - 128;               // 0 .. 255
    const int row = tid & 127;                       // query row of the unit = TMEM lane
    const uint32_t lanes = (uint32_t)(row & ~31) << 16;
    const uint32_t s_col = tmem + lanes + x * kColsS, o_col = tmem + lanes + kColO + x * 128;
    uint32_t ns = 0, npv = 0, nrot = 0, no = 0;      // parities (ns: one per buffer)
    int it = 0;                                      // blocks of the units before
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
      named_barrier_sync(1, 320);
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
        named_barrier_sync(1, 320);
      }
      const float bias = vis ? bias_s[row] : 0.f;
      RowStat st{-INFINITY, 0.f};
      const bool busy = (row & ~31) < live;          // some row of this warp exists
      const int nf = j0 < sp.blocks_full ? min(j1, sp.blocks_full) - j0 : 0;
      const int subs = nf + 2 * (j1 - j0 - nf);
      const int tok_vis = (max(j0, sp.blocks_full) - sp.blocks_full) * kVisTok;   // the segment's first visual token
      for (int i = x; i < subs; i += 2) {
        const int b = (i >> 1) & 1;
        const bool prompt = i < nf;
        const int tok = prompt ? (j0 + i) * kSub : tok_vis + (i - nf) * kSub;
        const int left = (prompt ? a.seq_full : a.seq_sparse) - tok;
        const bool masked = prompt && a.mask.data != nullptr;
        uint32_t v0 = ~0u, v1 = ~0u;
        if (masked || left < kSub) {
          const uint8_t *mk = static_cast<const uint8_t *>(a.mask.data) + pre * a.mask.s[0];
          v0 = __ballot_sync(0xffffffffu, lane < left && (!masked || mk[(tok + lane) * a.mask.s[1]] != 0));
          v1 = __ballot_sync(0xffffffffu, lane + 32 < left && (!masked || mk[(tok + lane + 32) * a.mask.s[1]] != 0));
        }
        const bool all = (v0 & v1) == ~0u;
        mbar_wait_bounded(&s_bar[x + 2 * b], (ns >> b) & 1, abort_flag, p.status);
        ns ^= 1u << b;
        tc_fence_after();
        if (masked && !all) {
          // a masked token's Values may hold anything, and 0 * NaN is NaN: zero them
          unsigned char *v = smem + L::kRing + (it + i) % L::kStages * L::kStage + 16384;
          for (int t = (warp & 3); t < kSub; t += 4)
            if (!(((t < 32 ? v0 : v1) >> (t & 31)) & 1u))
              *reinterpret_cast<uint2 *>(v + (lane >> 4) * 8192 + t * 128 + (lane & 15) * 8) = make_uint2(0, 0);
          fence_proxy_async_smem();
        }
        if (busy)
          softmax_sub<T>(s_col + 2 * b * kColsS, a.scale_log2, prompt ? 0.f : bias, all, v0, v1, st, [&](float f) {
            if (i < 2) return;                       // nothing in O yet
            // O is at rest once the P . V before this sub-block is done: the next S comes
            // after it in the tensor core's order; before the last one it is signalled
            if (i + 2 < subs)
              mbar_wait_bounded(&s_bar[x + 2 * (b ^ 1)], (ns >> (b ^ 1)) & 1, abort_flag, p.status);
            else
              mbar_wait_bounded(&pv_bar[x], npv, abort_flag, p.status);
            tc_fence_after();
            rescale_o(o_col, f);
          }, [&] {
            // The two streams' warps of a scheduler take turns with its exponential unit: while
            // one computes weights the other waits for S, reads it and finds its maximum
            // (left to themselves they run in step, and want the unit, and leave it idle, at
            // the same time: 490 -> 409 us for 4096 rows on 32,768 tokens of 8 heads).
            if (i > 0) named_barrier_sync(3 + (warp & 3) + 4 * (x ^ 1), 64);
          });
        if (busy && i + 1 < subs) asm volatile("bar.arrive %0, 64;" ::"r"(3 + (warp & 3) + 4 * x) : "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_bar[x + 2 * b]);
      }
      it += j1 - j0;
      if (subs > x + 2) npv ^= 1u;                   // one signal per unit whose stream has two sub-blocks
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
      const bool two = subs > 1;                     // the odd stream had a sub-block
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
      named_barrier_sync(1, 320);
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
  cudaError_t e = allow_shared_memory<shared_prefix_kernel<T, DK>>(smem);
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
