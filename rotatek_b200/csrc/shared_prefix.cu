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
//   P  = 2^(x - m) in two 16-bit parts, Phi + Plo; l sums it unrounded
//   O += Phi . V + Plo . V     (Phi alone would move outputs by 2^-9 of sum P |v|; the
//                       decode of one question per image splits its weights as well)
//
// m follows the running maximum lazily: O and l are rescaled only when a maximum
// grows by more than 2^8 over the one in use (P stays below 2^8, O and l are fp32).
//
// CTA (one per SM, 11 warps):
//   warps 0-3   softmax of the even blocks: thread = query row (TMEM lane)
//   warps 4-7   softmax of the odd blocks
//   warp 8      TMA producer: a ring of stages, one block's K and V each
//   warp 9      issues the MMAs of S (one elected lane); owns the TMEM
//   warp 10     issues those of O: a single thread's instructions could not keep the
//               tensor core fed
// TMEM (all 512 columns): three S buffers of 128, O of 128.  The S of the next blocks is made
// while two blocks are in the softmax; P goes over its S as the A operand of P . V, the upper
// 64 tokens first, whose P . V then begins.  The two softmax groups settle m in the order of the blocks, through
// shared memory; only where m moves does the group wait for the P . V before and rescale O.
// At the end of a unit the partial result of (unit, CTA) is written for shared_merge.cu.
//
// What bounds it: with many rows the tensor core (20 MMAs of 64 cycles a visual block, 16 of
// them P . V) and the exponential unit (128 x 128 a block at 16 a cycle: 1024 cycles), at the
// clocks that a sustained run is left with; with few rows, HBM and the latencies at a unit's ends.
//
// Measured: 4096 rows of each of 8 heads on 1024 + 31744 tokens 494 us (the tensor core alone
// 357, 421 at its sustained rate; the exponential unit 246); 560 rows, 4 prefixes of 4 heads on
// 640 + 15360 tokens 93; 12 rows, 2 prefixes of 32 heads on 32 + 16384 tokens 70 (344 MB); 56
// rows, 4 heads on 640 + 15360 tokens (111 SMs) 14.2; 14 rows, 4 heads on 64 + 1000 tokens 8.2.
// With one part of P these took 390, 82, 64, 13.4 and 8.0, with the P . V of a block begun only
// when all of its P was there (not its upper 64 tokens) 509, 96, 73, 14.4 and 8.3.
//
// Taken, and measured with one part of P for the first of these: 487 us before the two softmax groups
// took turns at the exponential unit, 409 after, P over S and one O so that a third S fits 400, the
// queries ahead of the ring 381.  Dropped: a sixth to a half of the exponentials as polynomials
// on the FMA units (378 to 404 where none took 373), three softmax groups (397), four that split
// a block's columns (402), blocks of 64 visual tokens (490 to 539).
#include <type_traits>

#include "shared.h"
#include "tcgen05.cuh"

namespace rtk {
namespace {

constexpr int kThreads = 352;
constexpr int kFullTok = 64, kVisTok = 128;      // tokens of a block
constexpr uint32_t kColsS = 128;                 // TMEM columns of an S buffer
// P over it: 64 tokens of S (64 columns) become 32 columns of Plo, then 32 of Phi
constexpr uint32_t kColHi = 32;
constexpr uint32_t kColO = 3 * kColsS;           // the O accumulator
constexpr float kLazy = 8.f;

// Where calls without a status word report a wait that gave up: zero when the library is
// loaded, so that a call that is being captured finds it ready.
__device__ unsigned int g_status;

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
  static constexpr int kRef = kDm + 512;                           // float[128]: m
  static constexpr int kMl = kRef + 512;                           // float2[2][128]: a group's m, l
  static constexpr int kBar = kMl + 2048;
  // full[S], empty[S], s_ready[3], p_ready[3], p_upper[3], pv_done[3], rot, o_done, q_here
  static constexpr int kNumBars = 2 * kStages + 15;
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
  tmem_wait_st();
}

// Columns [s, s + 64) of S whose token does not count become -inf, whatever was there.
__device__ __forceinline__ void mask_s(uint32_t s, uint32_t v0, uint32_t v1) {
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    const uint32_t v = (c < 2 ? v0 : v1) >> (16 * (c & 1));
    uint32_t r[16];
    tmem_ld16_nowait(s + 16 * c, r);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (!((v >> i) & 1u)) r[i] = 0xff800000u;
    tmem_st16_nowait(s + 16 * c, r);
  }
  tmem_wait_st();
}

__device__ __forceinline__ void load_half(uint32_t s, uint32_t (&r)[2][32]) {
  tmem_ld32_nowait(s, r[0]);
  tmem_ld32_nowait(s + 32, r[1]);
  tmem_wait_ld();
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

// Weights of the 64 columns at `p`: Plo and Phi (16-bit pairs) over them; returns their sum.
template <typename T>
__device__ __forceinline__ float weights_half(uint32_t p, const uint32_t (&r)[2][32], float scale, float off) {
  const float2 scale2 = make_float2(scale, scale), off2 = make_float2(off, off);
  float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t hi[16], lo[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float2 x = __ffma2_rn(make_float2(__uint_as_float(r[c][2 * i]), __uint_as_float(r[c][2 * i + 1])), scale2, off2);
      x.x = fast_exp2(x.x);
      x.y = fast_exp2(x.y);
      l2[i & 1] = __fadd2_rn(l2[i & 1], x);
      hi[i] = pack2<T>(x.x, x.y);
      float2 h;
      unpack2<T>(hi[i], h.x, h.y);
      x = __ffma2_rn(h, make_float2(-1.f, -1.f), x);       // exact
      lo[i] = pack2<T>(x.x, x.y);
    }
    tmem_st16_nowait(p + kColHi + 16 * c, hi);
    tmem_st16_nowait(p + 16 * c, lo);
  }
  return (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
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
  uint64_t *s_bar = empty_bar + L::kStages;       // [buffer] S is in TMEM
  uint64_t *p_bar = s_bar + 3;                    // [buffer] P is in TMEM
  uint64_t *up_bar = p_bar + 3;                   // [buffer] P of tokens 64 .. 127 is (prompt blocks: nothing)
  uint64_t *pv_bar = up_bar + 3;                  // [buffer] its P . V is done
  uint64_t *rot_bar = pv_bar + 3;                 // rotated queries are in TMEM
  uint64_t *o_bar = rot_bar + 1;                  // the O accumulator is complete
  uint64_t *q_bar = o_bar + 1;                    // the first unit's queries are here
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::kTmemSlot);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::kAbort);
  float *bias_s = reinterpret_cast<float *>(smem + L::kBias);
  float *dm_s = reinterpret_cast<float *>(smem + L::kDm);
  float *ref_s = reinterpret_cast<float *>(smem + L::kRef);
  float2 *ml_s = reinterpret_cast<float2 *>(smem + L::kMl);

  launch_dependents();
  const PrefixSplit &sp = p.split;
  const SharedParams &a = p.s;
  unsigned int *const status = p.status != nullptr ? p.status : &g_status;
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
    for (int i = 0; i < 3; ++i) {
      mbar_init(&s_bar[i], 1);
      mbar_init(&p_bar[i], 4);
      mbar_init(&up_bar[i], 4);
      mbar_init(&pv_bar[i], 1);
    }
    mbar_init(rot_bar, 1);
    mbar_init(o_bar, 1);
    mbar_init(q_bar, 8);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 8) {
    // ---------------------------------------------------------------- producer
    if (lane > 0) {
      // the queries and R of the CTA's later units, into L2 before they are asked for
      for (int u = u0 + 1; u <= u1; ++u) {
        const int ph = u / sp.row_tiles, pre = ph / a.kv_heads, h = ph % a.kv_heads;
        const int base = (u % sp.row_tiles) * 128, live = min(128, sp.rows - base);
        for (int e = lane - 1; e < 2 * live; e += 31) {
          const int r = base + (e >> 1), g = r % a.groups, nt = r / a.groups;
          prefetch_l2(static_cast<const T *>(a.q.data) + ((long long)pre * a.questions + nt / a.tokens) * a.q.s[0] +
                      (nt % a.tokens) * a.q.s[1] + (h * a.groups + g) * a.q.s[2] + (e & 1) * 64);
        }
        if (sp.blocks_vis > 0 && p.R_layout != 0) {
          const T *R = static_cast<const T *>(a.R.data) + pre * a.R.s[0] + h * a.R.s[1];
          if (p.R_layout == 1)
            for (int d = lane - 1; d < 128; d += 31) prefetch_l2(R + d * a.R.s[2]);
          else
            for (int e = lane - 1; e < 2 * DK; e += 31) prefetch_l2(R + (e >> 1) * a.R.s[3] + (e & 1) * 64);
        }
      }
    } else {
      int it = 0;
      bool ok = true;
      for (int u = u0; u <= u1 && ok; ++u) {
        const long long w = (long long)u * sp.unit_weight;
        const int j0 = r0 > w ? sp.block_from((int)(r0 - w)) : 0;
        const int j1 = r1 - w >= sp.unit_weight ? sp.blocks() : sp.block_from((int)(r1 - w));
        const int ph = u / sp.row_tiles, pre = ph / a.kv_heads, h = ph % a.kv_heads;
        for (int j = j0; j < j1; ++j, ++it) {
          const int stg = it % L::kStages;
          // one block ahead of the queries, the rest of the ring after them: every CTA's whole
          // ring would queue at HBM in front of them
          if (it == 1) mbar_wait_bounded(q_bar, 0, abort_flag, status);
          if (!mbar_wait_bounded(&empty_bar[stg], ((it / L::kStages) & 1) ^ 1, abort_flag, status)) {
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
          mbar_wait_bounded(&full_bar[k % L::kStages], (k / L::kStages) & 1, &dead, status);
      }
    }
  } else if (warp >= 9) {
    // ---------------------------------------------------------------- MMA issuers
    const bool for_s = warp == 9;
    constexpr uint32_t kFmt = kBf16 ? 1u : 0u;
    constexpr uint32_t kIdRot = idesc_f16(kFmt, 0, 0, 128, DK);
    constexpr uint32_t kIdFull = idesc_f16(kFmt, 0, 0, 128, kFullTok);
    constexpr uint32_t kIdVis = idesc_f16(kFmt, 0, 0, 128, kVisTok);
    constexpr uint32_t kIdPv = idesc_f16(kFmt, 0, 1, 128, 128);
    constexpr uint32_t kStep = L::kStage >> 4;       // from stage to stage, in a descriptor
    const uint32_t rot_addr = smem_u32(smem + L::kRot), ring = smem_u32(smem + L::kRing);
    const uint64_t q_desc = smem_desc_kmajor<128>(smem_u32(smem + L::kQ)), rot_desc = smem_desc_kmajor<128>(rot_addr);
    const uint64_t k_prompt = smem_desc_kmajor<128>(ring), v_prompt = smem_desc_sw128(ring + 16384, 8192, 1024);
    const uint64_t k_vis = smem_desc_kmajor<DK * 2>(ring), v_vis = smem_desc_sw128(ring + L::kKeyBytes, 16384, 1024);
    // stage and S buffer of the next block, and the parities of their rounds.  Issuing is
    // what the tensor core waits for, so they are carried along, not computed.
    uint32_t stage = 0, stage_par = 0, buf = 0, buf_par = 0;
    auto next = [&] {
      if (++stage == (uint32_t)L::kStages) {
        stage = 0;
        stage_par ^= 1u;
      }
      if (++buf == 3u) {
        buf = 0;
        buf_par ^= 1u;
      }
    };
    for (int u = u0; u <= u1; ++u) {
      const long long w = (long long)u * sp.unit_weight;
      const int j0 = r0 > w ? sp.block_from((int)(r0 - w)) : 0;
      const int j1 = r1 - w >= sp.unit_weight ? sp.blocks() : sp.block_from((int)(r1 - w));
      if (j0 >= j1) continue;
      named_barrier_sync(1, 320);            // Q and R^T are in shared memory
      if (j1 > sp.blocks_full) {
        if (for_s && elect_one()) {
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
        if (for_s) {
          for (int j = j0; j < j1; ++j) {
            // the buffer's last P has been used (the first round finds its parity done)
            mbar_wait_bounded(&pv_bar[buf], buf_par ^ 1u, abort_flag, status);
            mbar_wait_bounded(&full_bar[stage], stage_par, abort_flag, status);
            tc_fence_after();
            const uint32_t d = tmem + buf * kColsS;
            if (j >= sp.blocks_full) {
              constexpr int kSteps = DK / 16;
              const uint64_t kd = k_vis + stage * kStep;
#pragma unroll
              for (int k = 0; k < 2 * kSteps; ++k) {
                const int col = 16 * k;      // of [Qhi | Qlo]
                umma_f16_ss(d, rot_desc + (((col >> 6) * 16384 + (col & 63) * 2) >> 4),
                            kd + (((k % kSteps) * 32) >> 4), kIdVis, k > 0);
              }
            } else {
              const uint64_t kd = k_prompt + stage * kStep;
#pragma unroll
              for (int k = 0; k < 8; ++k)
                umma_f16_ss(d, q_desc + (((k >> 2) * 16384 + (k & 3) * 32) >> 4),
                            kd + (((k >> 2) * 8192 + (k & 3) * 32) >> 4), kIdFull, k > 0);
            }
            umma_commit(&s_bar[buf]);
            next();
          }
        } else {
          for (int j = j0; j < j1; ++j) {
            mbar_wait_bounded(&full_bar[stage], stage_par, abort_flag, status);
            mbar_wait_bounded(&up_bar[buf], buf_par, abort_flag, status);
            tc_fence_after();
            const uint32_t pa = tmem + buf * kColsS, first = j > j0;
            if (j >= sp.blocks_full) {
              const uint64_t vd = v_vis + stage * kStep;
#pragma unroll
              for (int k = 0; k < kVisTok / 16; ++k) {
                const int t = k ^ 4;                 // the upper tokens first
                if (k == 4) {
                  mbar_wait_bounded(&p_bar[buf], buf_par, abort_flag, status);
                  tc_fence_after();
                }
                const uint32_t pk = pa + (t >> 2) * 64 + (t & 3) * 8;
                umma_f16_ts(tmem + kColO, pk + kColHi, vd + ((t * 2048) >> 4), kIdPv, k > 0 ? 1u : first);
                umma_f16_ts(tmem + kColO, pk, vd + ((t * 2048) >> 4), kIdPv, 1u);
              }
            } else {
              mbar_wait_bounded(&p_bar[buf], buf_par, abort_flag, status);
              tc_fence_after();
              const uint64_t vd = v_prompt + stage * kStep;
#pragma unroll
              for (int k = 0; k < kFullTok / 16; ++k) {
                umma_f16_ts(tmem + kColO, pa + kColHi + 8 * k, vd + ((k * 2048) >> 4), kIdPv, k > 0 ? 1u : first);
                umma_f16_ts(tmem + kColO, pa + 8 * k, vd + ((k * 2048) >> 4), kIdPv, 1u);
              }
            }
            umma_commit(&pv_bar[buf]);
            umma_commit(&empty_bar[stage]);
            next();
          }
          umma_commit(o_bar);
        }
      }
      __syncwarp();
      named_barrier_sync(1, 320);            // the unit's partial has been read out
    }
  } else {
    // ---------------------------------------------------------------- softmax
    const int x = warp >> 2;                         // group: even or odd blocks of a unit
    const int tid = threadIdx.x;                     // 0 .. 255
    const int row = tid & 127;                       // query row of the unit = TMEM lane
    const uint32_t lanes = (uint32_t)(row & ~31) << 16;
    const uint32_t o_col = tmem + lanes + kColO;
    uint32_t nrot = 0, no = 0;                       // parities
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
        // queries: thread = half a row (8 chunks of 16 bytes).  Every load of the prologue is
        // in flight before the first is stored: beside the tiles' stream each round trip
        // takes microseconds.
        const int qrow = tid >> 1, half = tid & 1;
        const T *src = nullptr;
        if (qrow < live) {
          const int r = base + qrow, g = r % a.groups, nt = r / a.groups;
          src = static_cast<const T *>(a.q.data) + ((long long)pre * a.questions + nt / a.tokens) * a.q.s[0] +
                (nt % a.tokens) * a.q.s[1] + (h * a.groups + g) * a.q.s[2] + half * 64;
        }
        const T *R = static_cast<const T *>(a.R.data) + pre * a.R.s[0] + h * a.R.s[1];
        uint4 qv[8], rv[DK / 16];
        float dm = 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c)
          qv[c] = src != nullptr ? __ldg(reinterpret_cast<const uint4 *>(src) + c) : make_uint4(0, 0, 0, 0);
        if (vis) {
#pragma unroll
          for (int i = 0; i < DK / 16; ++i) {
            const int e = tid + 256 * i;
            if (p.R_layout == 1)                       // rows of R, 8 columns at a time
              rv[i] = __ldg(reinterpret_cast<const uint4 *>(R + (e / (DK / 8)) * a.R.s[2] + (e % (DK / 8)) * 8));
            else if (p.R_layout == 2)                  // columns of R, 8 rows at a time
              rv[i] = __ldg(reinterpret_cast<const uint4 *>(R + (e >> 4) * a.R.s[3] + (e & 15) * 8));
          }
          if (tid < 128 && a.dm.data != nullptr)
            dm = to_f32(static_cast<const T *>(a.dm.data)[pre * a.dm.s[0] + h * a.dm.s[1] + tid]);
        }
        unsigned char *dst = smem + L::kQ + half * 16384;
#pragma unroll
        for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4 *>(dst + swizzled_offset<128>(qrow, c * 8)) = qv[c];
        if (vis) {
          // R^T, K-major: row j holds column j of R
          const uint32_t rt = smem_u32(smem + L::kRot);
          if (p.R_layout == 0) {                       // any strides
#pragma unroll 8
            for (int e = tid; e < 128 * DK; e += 256) {
              const int d = e & 127, j = e >> 7;
              st_shared_u16(rt + (d >> 6) * (DK * 128) + swizzled_offset<128>(j, (d & 63) & ~7) + (d & 7) * 2,
                            __ldg(reinterpret_cast<const unsigned short *>(R + d * a.R.s[2] + j * a.R.s[3])));
            }
          } else {
#pragma unroll
            for (int i = 0; i < DK / 16; ++i) {
              const int e = tid + 256 * i;
              if (p.R_layout == 1) {
                const int d = e / (DK / 8), c = e % (DK / 8);
                const uint32_t words[4] = {rv[i].x, rv[i].y, rv[i].z, rv[i].w};
                const uint32_t box = rt + (d >> 6) * (DK * 128);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  st_shared_u16(box + swizzled_offset<128>(c * 8 + k, (d & 63) & ~7) + (d & 7) * 2,
                                (uint16_t)(words[k >> 1] >> (16 * (k & 1))));
              } else {
                const int j = e >> 4, c = e & 15;
                st_shared_v4(rt + (c >> 3) * (DK * 128) + swizzled_offset<128>(j, (c & 7) * 8), rv[i].x, rv[i].y, rv[i].z,
                             rv[i].w);
              }
            }
          }
          if (tid < 128) dm_s[tid] = dm;
        }
      }
      if (it == 0) {                                   // the first unit of this CTA
        __syncwarp();
        if (lane == 0) mbar_arrive(q_bar);
      }
      fence_proxy_async_smem();
      named_barrier_sync(1, 320);
      if (vis) {
        if (x == 0) {
          // rotated queries out of TMEM, as two 16-bit parts into shared memory
          mbar_wait_bounded(rot_bar, nrot & 1, abort_flag, status);
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
      float m = -INFINITY, l = 0.f;                  // what this group's last weights were relative to; their sum
      const bool busy = (row & ~31) < live;          // some row of this warp exists
      const int blocks = j1 - j0;
      for (int k = x; k < blocks; k += 2) {
        const int j = j0 + k, buf = (it + k) % 3;
        const uint32_t par = ((it + k) / 3) & 1;
        const bool prompt = j < sp.blocks_full;
        const int left = prompt ? a.seq_full - j * kFullTok : a.seq_sparse - (j - sp.blocks_full) * kVisTok;
        const bool masked = prompt && a.mask.data != nullptr;
        uint32_t v0 = ~0u, v1 = ~0u;
        if (masked) {
          const uint8_t *mk = static_cast<const uint8_t *>(a.mask.data) + pre * a.mask.s[0];
          const long long tok = j * kFullTok + lane;
          v0 = __ballot_sync(0xffffffffu, lane < left && mk[tok * a.mask.s[1]] != 0);
          v1 = __ballot_sync(0xffffffffu, lane + 32 < left && mk[(tok + 32) * a.mask.s[1]] != 0);
        }
        mbar_wait_bounded(&s_bar[buf], par, abort_flag, status);
        tc_fence_after();
        const uint32_t s = tmem + lanes + buf * kColsS;
        if (masked && (v0 & v1) != ~0u) {
          // a masked token's Values may hold anything, and 0 * NaN is NaN: zero them
          unsigned char *v = smem + L::kRing + (it + k) % L::kStages * L::kStage + 16384;
          for (int t = (warp & 3); t < kFullTok; t += 4)
            if (!(((t < 32 ? v0 : v1) >> (t & 31)) & 1u))
              *reinterpret_cast<uint2 *>(v + (lane >> 4) * 8192 + t * 128 + (lane & 15) * 8) = make_uint2(0, 0);
          fence_proxy_async_smem();
          mask_s(s, v0, v1);
        } else if (left < (prompt ? kFullTok : kVisTok)) {
          auto bits = [&](int n) { return n >= 32 ? ~0u : n > 0 ? (1u << n) - 1u : 0u; };
          mask_s(s, bits(left), bits(left - 32));
          if (!prompt) mask_s(s + 64, bits(left - 64), bits(left - 96));
        }
        if (busy) {
          uint32_t r[2][32];
          load_half(s, r);
          float mx = max_half(r);
          if (!prompt) {                             // the upper half stays in registers
            load_half(s + 64, r);
            mx = fmaxf(mx, max_half(r));
          }
          const float bi = prompt ? 0.f : bias;
          const float top = fmaf(mx, a.scale_log2, bi);     // scale > 0; -inf stays -inf
          // m, as the block before has settled it
          float now = -INFINITY;
          if (k > 0) {
            named_barrier_sync(3 + (warp & 3) + 4 * (x ^ 1), 64);
            now = ref_s[row];
          }
          const bool grow = top > now + kLazy;       // from -inf: whenever there is a maximum
          if (__any_sync(0xffffffffu, grow)) {
            const float f = grow ? fast_exp2(now - top) : 1.f;      // first maximum: 2^-inf = 0
            if (grow) now = top;
            if (k > 0) {                             // O is at rest when the P . V before is done
              const int g = it + k - 1;
              mbar_wait_bounded(&pv_bar[g % 3], (g / 3) & 1, abort_flag, status);
              tc_fence_after();
              rescale_o(o_col, f);
              tc_fence_before();
            }
            ref_s[row] = now;
          } else if (k == 0) {
            ref_s[row] = now;
          }
          if (k + 1 < blocks) asm volatile("bar.arrive %0, 64;" ::"r"(3 + (warp & 3) + 4 * x) : "memory");
          if (__any_sync(0xffffffffu, m != now)) {   // the other group moves it too
            l *= m > -INFINITY ? fast_exp2(m - now) : 0.f;
            m = now;
          }
          const float off = bi - (m > -INFINITY ? m : 0.f);
          if (!prompt) {
            l += weights_half<T>(s + 64, r, a.scale_log2, off);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&up_bar[buf]);
            load_half(s, r);
          }
          l += weights_half<T>(s, r, a.scale_log2, off);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (prompt || !busy) mbar_arrive(&up_bar[buf]);
          mbar_arrive(&p_bar[buf]);
        }
      }
      it += blocks;
      // the partial result: each group writes 64 channels of the row
      ml_s[x * 128 + row] = make_float2(m, l);
      mbar_wait_bounded(o_bar, no & 1, abort_flag, status);
      ++no;
      tc_fence_after();
      named_barrier_sync(2, 256);
      const long long slot = u + cta;
      if (busy) {
        const float ref = ref_s[row];
        // four channels of a row together, rows side by side: a warp's stores are whole lines
        float4 *out = reinterpret_cast<float4 *>(p.acc) + (slot * 32 + 16 * x) * 128 + row;
#pragma unroll
        for (int c = 0; c < 64; c += 16) {
          uint32_t r[16];
          tmem_ld16_nowait(o_col + 64 * x + c, r);
          tmem_wait_ld();
          if (row < live) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              out[(c / 4 + i) * 128] = make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]),
                                                   __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
          }
        }
        if (x == 0 && row < live) {
          float sum = 0.f;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const float2 e = ml_s[g * 128 + row];
            sum = fmaf(e.y, e.x > -INFINITY ? fast_exp2(e.x - ref) : 0.f, sum);
          }
          // a row whose logits are NaN stays one: m NaN, as no weight may drop it
          reinterpret_cast<float2 *>(p.ml)[slot * 128 + row] = make_float2(isnan(sum) ? sum : ref, sum);
        }
      }
      tc_fence_before();
      named_barrier_sync(1, 320);
    }
  }
  __syncthreads();
  if (warp == 9) {
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

cudaError_t shared_status_address(void **address) { return cudaGetSymbolAddress(address, g_status); }

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
