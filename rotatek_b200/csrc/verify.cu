// Verification of drafted tokens against the target model, from random numbers
// that the caller gives.
//
// For question b with n = draft_lens[b] drafts x_0 .. x_{n-1} and temperature h:
//   h > 0   p_j = softmax(target[b, j] / h), q_j = softmax(draft[b, j] / h) (one-hot at
//           x_j without draft logits); draft j is accepted when u_j q_j(x_j) < p_j(x_j)
//           and all before it were.  With k drafts accepted the next token is
//               argmax_i w_i / e_i,   w = max(p_k - q_k, 0) if k < n, else p_k
//           (w = p_k too where the difference leaves nothing), lowest index on ties.
//           With e_i ~ Exp(1) the smallest e_i / w_i is token i with probability
//           w_i / sum w: an exponential race draws from the normalised residual without
//           a cumulative sum, so the answer does not depend on an order of summation.
//   h <= 0  draft j is accepted when it is argmax target[b, j] (lowest index); the
//           next token is the argmax of row k.
//
// Two kernels.  stats: a CTA per (row, chunk of the vocabulary) leaves the chunk's
// maximum and sum of exponentials relative to it (a greedy row: its maximum and where): one
// pass over every logits row that a decision can read, in 16-byte loads.
// pick: a cluster of up to 8 CTAs per question joins the rows' chunks (a warp per row, always
// in the same tree), finds k, and races over row k alone, which the first pass left in L2 or
// near it; the CTAs' winners, 64-bit keys (value, ~index), meet in the shared memory of the
// first.  (Through atomics in device memory the end took 1.2 us longer.)  pick is launched
// while stats still runs and waits for it on the device.
//
// Measured, and what bounds it: 128 questions, up to 8 drafts, 131071 bf16 logits, 251 MB in
// 62.9 us: stats 39 at 4.7 TB/s (the exponential unit alone needs half of that), then
// 22 for the race, which reads the noise for the first time.  64 questions, up to 5 drafts,
// 32000 fp16 logits of both models, 37 MB: 20.0 us, 10 each.  One question: 9.6 us, the
// latency of two dependent kernels.
#include <type_traits>

#include "common.cuh"
#include "shared.h"

namespace rtk {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDrafts = 64;
constexpr float kLog2e = 1.4426950408889634f;

struct VerifyLayout {
  int chunk, chunks;           // vocabulary elements of a chunk, chunks of a row (stats)
  int race, races;             // the same of the race (pick)
  int rows;                    // logits rows of a question: 2 T + 1
};

// Chunks of at least 2048 elements (a 16-byte load of each thread), larger where there
// are enough rows to fill the SMs several times over: what a CTA does before and after its
// loads is paid per chunk (the 251 MB above: 199 us with 2048, 67 with 16384, 63 with 65536;
// 37 MB: 32 and 20).
__host__ __device__ inline VerifyLayout verify_layout(long long batch, long long drafts, long long vocab) {
  VerifyLayout l;
  l.rows = (int)(2 * drafts + 1);
  const long long total = batch * l.rows * vocab;
  l.chunk = 2048;
  while (l.chunk < 65536 && total / l.chunk > 148 * 16) l.chunk *= 2;
  l.chunks = (int)((vocab + l.chunk - 1) / l.chunk);
  // pick: one wave of CTAs, since each of them joins and decides before it races (two waves:
  // 67.5 against 62.9 us at 128 questions); a cluster of 1, 2, 4 or 8 per question (one
  // question: 10.3 us with 4, 9.0 with 8)
  l.races = 8;
  while (l.races > 1 && (batch * l.races > 148 * 4 || vocab < 1024 * l.races)) l.races /= 2;
  l.race = (int)((vocab + l.races * 64 - 1) / (l.races * 64) * 64);
  return l;
}

// The workspace holds float4 (max, sum, argmax bits, -) per (b, row, chunk).

__device__ __forceinline__ int drafts_of(const VerifyParams &p, int b) {
  return p.draft_lens != nullptr ? min(max(p.draft_lens[b * p.dl_s], 0), p.drafts) : p.drafts;
}

// logits row r of question b: rows 0 .. T the target's, T + 1 .. 2 T the draft's
template <typename T>
__device__ __forceinline__ const T *logits_row(const VerifyParams &p, int b, int r) {
  return r <= p.drafts ? static_cast<const T *>(p.target.data) + b * p.target.s[0] + r * p.target.s[1]
                       : static_cast<const T *>(p.draft.data) + b * p.draft.s[0] + (r - p.drafts - 1) * p.draft.s[1];
}

// 2^((x - m) c): the difference is taken first, since x c and m c of a tiny temperature are too large for
// theirs to mean anything
__device__ __forceinline__ float weight(float x, float m, float c) { return fast_exp2((x - m) * c); }

// (m, z): a maximum and the sum of weights relative to it; c = log2(e) / temperature
__device__ __forceinline__ void join(float &m, float &z, float m2, float z2, float c) {
  const float top = fmaxf(m, m2);
  if (top == -INFINITY) return;                  // nothing on either side
  z = z * weight(m, top, c) + z2 * weight(m2, top, c);
  m = top;
}

// packed (value, lowest index wins): values are >= 0, so their bits order them
__device__ __forceinline__ unsigned long long race_key(float v, unsigned i) {
  return ((unsigned long long)__float_as_uint(v) << 32) | (0xffffffffu - i);
}

// The chunk [i0, i1) of a row as visited by this thread: f(first index, n, values) with n
// values at consecutive indices, ascending.  Whole aligned 16-byte words are loaded as
// such, four of a thread in flight; what lies before and after them one by one.
template <typename T, typename F>
__device__ __forceinline__ void visit(const T *row, int i0, int i1, F f) {
  constexpr int kVec = 16 / sizeof(T);
  const int off = (int)((reinterpret_cast<uintptr_t>(row + i0) / sizeof(T)) % kVec);
  const int head = min(i1 - i0, off ? kVec - off : 0);
  const int words = (i1 - i0 - head) / kVec, tail = i0 + head + words * kVec;
  float one[kVec];
  if ((int)threadIdx.x < head) {
    one[0] = to_f32(row[i0 + threadIdx.x]);
    f(i0 + (int)threadIdx.x, 1, one);
  }
  const uint4 *body = reinterpret_cast<const uint4 *>(row + i0 + head);
  for (int w = threadIdx.x; w < words; w += 4 * kThreads) {
    uint4 raw[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (w + k * kThreads < words) raw[k] = __ldg(body + w + k * kThreads);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (w + k * kThreads >= words) break;
      const uint32_t u[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
      float v[kVec];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 4) v[e] = __uint_as_float(u[e]);
        else unpack2<T>(u[e], v[2 * e], v[2 * e + 1]);
      }
      f(i0 + head + (w + k * kThreads) * kVec, kVec, v);
    }
  }
  if (tail + (int)threadIdx.x < i1) {
    one[0] = to_f32(row[tail + threadIdx.x]);
    f(tail + (int)threadIdx.x, 1, one);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_stats_kernel(const VerifyParams p) {
  __shared__ float m_s[kThreads / 32], z_s[kThreads / 32];
  __shared__ int i_s[kThreads / 32];
  launch_dependents();
  const VerifyLayout l = verify_layout(p.batch, p.drafts, p.vocab);
  const int r = blockIdx.y, b = blockIdx.z, chunk = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = drafts_of(p, b);
  const float heat = p.temperature[b * p.temp_s];
  const bool greedy = !(heat > 0.f);
  const bool is_draft = r > p.drafts;
  if (is_draft ? (greedy || r - p.drafts - 1 >= n) : r > n) return;   // a row that no decision reads
  const T *row = logits_row<T>(p, b, r);
  const int i0 = chunk * l.chunk, i1 = min(p.vocab, i0 + l.chunk);
  float m = -INFINITY, z = 0.f;                // the maximum logit; sum 2^((x - m) c)
  int at = i0;
  const float c = greedy ? 1.f : kLog2e / fmaxf(heat, 1e-30f);
  if (greedy) {
    visit<T>(row, i0, i1, [&](int i, int cnt, const float *v) {
#pragma unroll
      for (int e = 0; e < 16 / (int)sizeof(T); ++e)
        if (e < cnt && (v[e] > m || (v[e] == m && i + e < at))) {
          m = v[e];
          at = i + e;
        }
    });
  } else {
    visit<T>(row, i0, i1, [&](int, int cnt, const float *v) {
      constexpr int kVec = 16 / sizeof(T);
      if (cnt == kVec) {
        float top = v[0];
#pragma unroll
        for (int e = 1; e < kVec; ++e) top = fmaxf(top, v[e]);
        if (top > m) {
          z *= weight(m, top, c);              // nothing yet: 0
          m = top;
        }
        if (m > -INFINITY) {
          const float2 from = make_float2(-m, -m), c2 = make_float2(c, c);
#pragma unroll
          for (int e = 0; e < kVec; e += 2) {
            const float2 x = __fmul2_rn(__fadd2_rn(make_float2(v[e], v[e + 1]), from), c2);
            z += fast_exp2(x.x) + fast_exp2(x.y);
          }
        }
      } else {
        if (v[0] > m) {
          z *= weight(m, v[0], c);
          m = v[0];
        }
        if (m > -INFINITY) z += weight(v[0], m, c);
      }
    });
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), z2 = __shfl_xor_sync(0xffffffffu, z, o);
    const int at2 = __shfl_xor_sync(0xffffffffu, at, o);
    if (greedy) {
      if (m2 > m || (m2 == m && at2 < at)) {
        m = m2;
        at = at2;
      }
    } else {
      join(m, z, m2, z2, c);
    }
  }
  if (lane == 0) {
    m_s[warp] = m;
    z_s[warp] = z;
    i_s[warp] = at;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) {
      if (greedy) {
        if (m_s[w] > m || (m_s[w] == m && i_s[w] < at)) {
          m = m_s[w];
          at = i_s[w];
        }
      } else {
        join(m, z, m_s[w], z_s[w], c);
      }
    }
    static_cast<float4 *>(p.workspace)[((long long)b * l.rows + r) * l.chunks + chunk] = make_float4(m, z, __int_as_float(at), 0.f);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) verify_pick_kernel(const VerifyParams p) {
  __shared__ float m_s[2 * kMaxDrafts + 1], z_s[2 * kMaxDrafts + 1];     // maximum, 1 / sum
  __shared__ int at_s[kMaxDrafts + 1];
  __shared__ int k_s;
  __shared__ unsigned long long key_s[kThreads / 32];
  __shared__ unsigned long long race_s[8];       // of the cluster's first CTA: every CTA's winner
  const VerifyLayout l = verify_layout(p.batch, p.drafts, p.vocab);
  const int b = blockIdx.y, chunk = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = drafts_of(p, b), T1 = p.drafts + 1;
  const float heat = p.temperature[b * p.temp_s];
  const bool greedy = !(heat > 0.f), soft_draft = p.draft.data != nullptr;
  const float c = greedy ? 1.f : kLog2e / fmaxf(heat, 1e-30f);
  if (greedy && chunk > 0) return;               // a greedy question's first CTA meets no barrier either
  const bool clustered = l.races > 1 && !greedy;
  if (clustered) cluster_arrive();               // this CTA has started: its shared memory is there
  const int i0 = chunk * l.race, i1 = min(p.vocab, i0 + l.race);
  const float *noise = p.noise + b * p.noise_s;
  // what an acceptance needs besides the sums: a draft per thread
  const int j = threadIdx.x;
  long long x = -1;
  float u = 0.f, tx = 0.f, dx = 0.f;
  if (j < n) {
    x = p.tokens[b * p.tok_s[0] + j * p.tok_s[1]];
    u = p.uniforms[b * p.uni_s[0] + j * p.uni_s[1]];
    if (x >= 0 && x < p.vocab && !greedy) {
      tx = to_f32(logits_row<T>(p, b, j)[x]);
      if (soft_draft) dx = to_f32(logits_row<T>(p, b, T1 + j)[x]);
    }
  }
  if (threadIdx.x == 0) k_s = n;
  wait_for_previous();

  // join the chunks of every row a decision may read: a warp per row
  for (int r = warp; r < l.rows; r += kThreads / 32) {
    const bool is_draft = r > p.drafts;
    if (is_draft ? (greedy || !soft_draft || r - T1 >= n) : r > n) continue;
    const float4 *st = static_cast<const float4 *>(p.workspace) + ((long long)b * l.rows + r) * l.chunks;
    float m = -INFINITY, z = 0.f;
    int at = 0x7fffffff;
    for (int i = lane; i < l.chunks; i += 32) {
      const float4 v = __ldcg(st + i);
      if (greedy) {
        if (v.x > m || (v.x == m && __float_as_int(v.z) < at)) {
          m = v.x;
          at = __float_as_int(v.z);
        }
      } else {
        join(m, z, v.x, v.y, c);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), z2 = __shfl_xor_sync(0xffffffffu, z, o);
      const int at2 = __shfl_xor_sync(0xffffffffu, at, o);
      if (greedy) {
        if (m2 > m || (m2 == m && at2 < at)) {
          m = m2;
          at = at2;
        }
      } else {
        join(m, z, m2, z2, c);
      }
    }
    if (lane == 0) {
      m_s[r] = m;
      z_s[r] = z > 0.f ? 1.f / z : 0.f;
      if (!is_draft) at_s[r] = at;
    }
  }
  __syncthreads();
  // p (or q) of a token of row r
  auto prob = [&](float m, float inv, float logit) {
    return m > -INFINITY ? weight(logit, m, c) * inv : 0.f;
  };
  if (j < n) {
    bool ok = false;
    if (x >= 0 && x < p.vocab) {                    // anything else is no token: rejected
      if (greedy) ok = x == at_s[j];
      else ok = u * (soft_draft ? prob(m_s[T1 + j], z_s[T1 + j], dx) : 1.f) < prob(m_s[j], z_s[j], tx);
    }
    if (!ok) atomicMin(&k_s, j);
  }
  __syncthreads();
  const int k = k_s;
  const bool rejected = k < n;
  const T *tr = logits_row<T>(p, b, k);
  const T *dr = rejected && soft_draft ? logits_row<T>(p, b, T1 + k) : nullptr;
  const long long gone = rejected && !soft_draft ? p.tokens[b * p.tok_s[0] + k * p.tok_s[1]] : -1;
  const int drop = gone >= 0 && gone < p.vocab ? (int)gone : -1;
  const float mt = m_s[k], zt = z_s[k], md = dr != nullptr ? m_s[T1 + k] : 0.f, zd = dr != nullptr ? z_s[T1 + k] : 0.f;
  // The best runner of [from, to).  About ten instructions a token: without a draft's logits
  // 1 / z is left out (it scales every runner alike), and a runner's index is looked up only
  // where a group of kU holds a new best.
  constexpr int kU = 8;
  auto race = [&](int from, int to, bool rest) {
    float top = 0.f;
    int who = 0;
    const bool minus = rest && dr != nullptr;
    const float ft = mt > -INFINITY ? mt : INFINITY, fd = md > -INFINITY ? md : INFINITY;      // nothing there: 2^-inf
    auto group = [&](int i, auto whole) {
      float t[kU], v[kU];
#pragma unroll
      for (int q = 0; q < kU; ++q) {
        const bool in = whole || i + q * kThreads < to;
        t[q] = in ? to_f32(tr[i + q * kThreads]) : -INFINITY;
        v[q] = in ? __ldg(noise + i + q * kThreads) : 1.f;
      }
      if (minus) {
        float d[kU];
#pragma unroll
        for (int q = 0; q < kU; ++q)
          d[q] = whole || i + q * kThreads < to ? to_f32(dr[i + q * kThreads]) : -INFINITY;
#pragma unroll
        for (int q = 0; q < kU; ++q)
          v[q] = __fdividef(__fsub_rn(__fmul_rn(weight(t[q], ft, c), zt),      // not fused:
                                      __fmul_rn(weight(d[q], fd, c), zd)),     // p - p is 0
                            v[q]);
      } else {
#pragma unroll
        for (int q = 0; q < kU; ++q) v[q] = __fdividef(weight(t[q], ft, c), v[q]);
        // a draft without logits is certain of its token: nothing of p is left there
        if (rest && (unsigned)(drop - i) <= (kU - 1) * kThreads && (drop - i) % kThreads == 0) {
#pragma unroll
          for (int q = 0; q < kU; ++q)
            if (i + q * kThreads == drop) v[q] = 0.f;
        }
      }
      float best = v[0];
#pragma unroll
      for (int q = 1; q < kU; ++q) best = fmaxf(best, v[q]);
      if (best > top) {                             // groups ascend: ties keep the lowest index
        top = best;
#pragma unroll
        for (int q = kU - 1; q >= 0; --q)
          if (v[q] == best) who = i + q * kThreads;
      }
    };
    int i = from + (int)threadIdx.x;
    for (; i + (kU - 1) * kThreads < to; i += kU * kThreads) group(i, std::true_type{});
    if (i < to) group(i, std::false_type{});
    unsigned long long best = top > 0.f ? race_key(top, (unsigned)who) : 0ull;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) key_s[warp] = best;
    __syncthreads();
    best = key_s[0];
    for (int w = 1; w < kThreads / 32; ++w) best = max(best, key_s[w]);
    return best;
  };
  long long next = at_s[greedy ? k : 0];
  if (!greedy) {
    unsigned long long key = race(i0, i1, rejected);
    if (clustered) {                               // the winners meet in the first CTA
      cluster_wait();
      if (threadIdx.x == 0) st_cluster_u64(&race_s[chunk], 0, key);
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      if (chunk > 0) return;
      for (int w = 1; w < l.races; ++w) key = max(key, race_s[w]);
    }
    if (key == 0ull && rejected) {                 // p - q left nothing: draw from p
      __syncthreads();
      key = race(0, p.vocab, false);
    }
    next = key == 0ull ? 0 : (long long)(0xffffffffu - (unsigned)(key & 0xffffffffull));
  }
  for (int i = threadIdx.x; i < T1; i += kThreads)
    p.out_tokens[(long long)b * T1 + i] = i < k ? p.tokens[b * p.tok_s[0] + i * p.tok_s[1]] : i == k ? next : -1ll;
  if (threadIdx.x == 0) p.accepted[b] = k;
}

template <typename T>
cudaError_t verify(const VerifyParams &p, cudaStream_t stream) {
  const VerifyLayout l = verify_layout(p.batch, p.drafts, p.vocab);
  const int rows = p.draft.data != nullptr ? l.rows : p.drafts + 1;
  verify_stats_kernel<T><<<dim3(l.chunks, rows, p.batch), kThreads, 0, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return launch_overlapping_clusters(verify_pick_kernel<T>, dim3(l.races, p.batch), dim3(kThreads), l.races, 0, stream, p);
}

}  // namespace

size_t verify_workspace_bytes(long long batch, long long drafts, long long vocab) {
  const VerifyLayout l = verify_layout(batch, drafts, vocab);
  return (size_t)(batch * l.rows * l.chunks * 16);
}

cudaError_t launch_verify(const VerifyParams &p, cudaStream_t stream) {
  if (p.batch == 0) return cudaSuccess;
  if (p.dtype == 0) return verify<float>(p, stream);
  if (p.dtype == 1) return verify<__nv_bfloat16>(p, stream);
  return verify<__half>(p, stream);
}

}  // namespace rtk
