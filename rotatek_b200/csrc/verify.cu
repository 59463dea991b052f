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
// running maximum and sum of exponentials (a greedy row: its maximum and where) --
// one pass over every logits row.  pick: CTAs per (question, chunk) join a row's
// chunks in chunk order, find k, and race over row k alone; the winners of the
// chunks meet in a 64-bit atomicMax on (value, ~index), whose result does not depend
// on the order of arrival.
#include "common.cuh"
#include "shared.h"

namespace rtk {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDrafts = 64;
constexpr float kLog2e = 1.4426950408889634f;

struct VerifyLayout {
  int chunk, chunks;           // vocabulary elements of a chunk, chunks of a row
  long long rows;              // logits rows of a question: 2 T + 1
};

__host__ __device__ inline VerifyLayout verify_layout(long long drafts, long long vocab) {
  VerifyLayout l;
  l.chunk = 8192;
  l.chunks = (int)((vocab + l.chunk - 1) / l.chunk);
  l.rows = 2 * drafts + 1;
  return l;
}

// workspace: [B] race keys (residual), [B] race keys (p), [B] tickets, then
// float4 (max, sum, argmax bits, -) per (b, row, chunk)
struct VerifySpace {
  unsigned long long *rest_key, *p_key;
  unsigned int *ticket;
  float4 *stats;
};

__host__ __device__ inline long long align16(long long x) { return (x + 15) / 16 * 16; }

__host__ __device__ inline VerifySpace verify_space(void *ws, long long batch) {
  VerifySpace s;
  unsigned char *p = static_cast<unsigned char *>(ws);
  s.rest_key = reinterpret_cast<unsigned long long *>(p);
  s.p_key = s.rest_key + batch;
  s.ticket = reinterpret_cast<unsigned int *>(s.p_key + batch);
  s.stats = reinterpret_cast<float4 *>(p + align16(batch * 20));
  return s;
}

__device__ __forceinline__ int drafts_of(const VerifyParams &p, int b) {
  return p.draft_lens != nullptr ? min(max(p.draft_lens[b * p.dl_s], 0), p.drafts) : p.drafts;
}

// logits row r of question b: rows 0 .. T the target's, T + 1 .. 2 T the draft's
template <typename T>
__device__ __forceinline__ const T *logits_row(const VerifyParams &p, int b, int r) {
  return r <= p.drafts ? static_cast<const T *>(p.target.data) + b * p.target.s[0] + r * p.target.s[1]
                       : static_cast<const T *>(p.draft.data) + b * p.draft.s[0] + (r - p.drafts - 1) * p.draft.s[1];
}

__device__ __forceinline__ void join(float &m, float &z, float m2, float z2) {
  const float top = fmaxf(m, m2);
  if (top == -INFINITY) return;                  // nothing on either side
  z = z * exp2f(m - top) + z2 * exp2f(m2 - top);
  m = top;
}

// packed (value, lowest index wins): values are >= 0, so their bits order them
__device__ __forceinline__ unsigned long long race_key(float v, unsigned i) {
  return ((unsigned long long)__float_as_uint(v) << 32) | (0xffffffffu - i);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_stats_kernel(const VerifyParams p) {
  __shared__ float m_s[kThreads / 32], z_s[kThreads / 32];
  __shared__ int i_s[kThreads / 32];
  const VerifyLayout l = verify_layout(p.drafts, p.vocab);
  const VerifySpace ws = verify_space(p.workspace, p.batch);
  const int r = blockIdx.y, b = blockIdx.z, chunk = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (r == 0 && chunk == 0 && threadIdx.x == 0) {
    ws.rest_key[b] = 0ull;
    ws.p_key[b] = 0ull;
    ws.ticket[b] = 0u;
  }
  const int n = drafts_of(p, b);
  const float heat = p.temperature[b * p.temp_s];
  const bool greedy = !(heat > 0.f);
  const bool is_draft = r > p.drafts;
  if (is_draft ? (greedy || r - p.drafts - 1 >= n) : r > n) return;   // a row that no decision reads
  const T *row = logits_row<T>(p, b, r);
  const int i0 = chunk * l.chunk, i1 = min(p.vocab, i0 + l.chunk);
  // base-2 logits relative to a running maximum, x = logit * log2(e) / h
  const float c = greedy ? 1.f : kLog2e / fmaxf(heat, 1e-30f);
  float m = -INFINITY, z = 0.f;
  int at = i0;
  for (int i = i0 + (int)threadIdx.x; i < i1; i += kThreads) {
    const float x = to_f32(row[i]) * c;
    if (greedy) {
      if (x > m) {
        m = x;
        at = i;
      }
    } else if (x > m) {
      z = fmaf(z, exp2f(m - x), 1.f);
      m = x;
    } else if (m > -INFINITY) {
      z += exp2f(x - m);
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
      join(m, z, m2, z2);
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
        join(m, z, m_s[w], z_s[w]);
      }
    }
    ws.stats[((long long)b * l.rows + r) * l.chunks + chunk] = make_float4(m, z, __int_as_float(at), 0.f);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_pick_kernel(const VerifyParams p) {
  __shared__ float m_s[2 * kMaxDrafts + 1], z_s[2 * kMaxDrafts + 1];
  __shared__ int at_s[kMaxDrafts + 1];
  __shared__ int k_s;
  __shared__ bool last_s;
  __shared__ unsigned long long rest_s[kThreads / 32], pk_s[kThreads / 32];
  const VerifyLayout l = verify_layout(p.drafts, p.vocab);
  const VerifySpace ws = verify_space(p.workspace, p.batch);
  const int b = blockIdx.y, chunk = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = drafts_of(p, b), T1 = p.drafts + 1;
  const float heat = p.temperature[b * p.temp_s];
  const bool greedy = !(heat > 0.f), soft_draft = p.draft.data != nullptr;
  if (greedy && chunk > 0) return;

  // join the chunks of every row a decision may read (in chunk order)
  for (int r = threadIdx.x; r < (int)l.rows; r += kThreads) {
    const bool is_draft = r > p.drafts;
    if (is_draft ? (greedy || !soft_draft || r - T1 >= n) : r > n) continue;
    const float4 *st = ws.stats + ((long long)b * l.rows + r) * l.chunks;
    float m = -INFINITY, z = 0.f;
    int at = 0;
    for (int i = 0; i < l.chunks; ++i) {
      const float4 v = st[i];
      if (greedy) {
        if (v.x > m) {                  // chunks come in index order: the first maximum stays
          m = v.x;
          at = __float_as_int(v.z);
        }
      } else {
        join(m, z, v.x, v.y);
      }
    }
    m_s[r] = m;
    z_s[r] = z;
    if (!is_draft) at_s[r] = at;
  }
  if (threadIdx.x == 0) k_s = n;
  __syncthreads();
  const float c = greedy ? 1.f : kLog2e / fmaxf(heat, 1e-30f);
  auto prob = [&](int r, float logit) {            // p (or q) of a token of row r
    return m_s[r] > -INFINITY ? exp2f(logit * c - m_s[r]) / z_s[r] : 0.f;
  };
  for (int j = threadIdx.x; j < n; j += kThreads) {
    const long long x = p.tokens[b * p.tok_s[0] + j * p.tok_s[1]];
    bool ok = false;
    if (x >= 0 && x < p.vocab) {                    // anything else is no token: rejected
      if (greedy) {
        ok = x == at_s[j];
      } else {
        const float pj = prob(j, to_f32(logits_row<T>(p, b, j)[x]));
        const float qj = soft_draft ? prob(T1 + j, to_f32(logits_row<T>(p, b, T1 + j)[x])) : 1.f;
        ok = p.uniforms[b * p.uni_s[0] + j * p.uni_s[1]] * qj < pj;
      }
    }
    if (!ok) atomicMin(&k_s, j);
  }
  __syncthreads();
  const int k = k_s;
  unsigned long long rest = 0ull, whole = 0ull;
  if (!greedy) {
    const T *tr = logits_row<T>(p, b, k);
    const bool rejected = k < n;
    const T *dr = rejected && soft_draft ? logits_row<T>(p, b, T1 + k) : nullptr;
    const long long drop = rejected && !soft_draft ? p.tokens[b * p.tok_s[0] + k * p.tok_s[1]] : -1;
    const float *e = p.noise + b * p.noise_s;
    const int i0 = chunk * l.chunk, i1 = min(p.vocab, i0 + l.chunk);
    for (int i = i0 + (int)threadIdx.x; i < i1; i += kThreads) {
      const float pi = prob(k, to_f32(tr[i]));
      const float ei = e[i];
      float w = pi;
      if (dr != nullptr) w = fmaxf(pi - prob(T1 + k, to_f32(dr[i])), 0.f);
      if (i == drop) w = fmaxf(pi - 1.f, 0.f);
      if (w > 0.f) rest = max(rest, race_key(w / ei, (unsigned)i));
      if (pi > 0.f) whole = max(whole, race_key(pi / ei, (unsigned)i));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      rest = max(rest, __shfl_xor_sync(0xffffffffu, rest, o));
      whole = max(whole, __shfl_xor_sync(0xffffffffu, whole, o));
    }
    if (lane == 0) {
      rest_s[warp] = rest;
      pk_s[warp] = whole;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kThreads / 32; ++w) {
        rest = max(rest, rest_s[w]);
        whole = max(whole, pk_s[w]);
      }
      atomicMax(&ws.rest_key[b], rest);
      atomicMax(&ws.p_key[b], whole);
      __threadfence();
      last_s = atomicAdd(&ws.ticket[b], 1u) == (unsigned)l.chunks - 1u;
    }
    __syncthreads();
    if (!last_s) return;
    __threadfence();
  }
  // the question's last CTA writes the answer
  long long next = at_s[greedy ? k : 0];
  if (!greedy) {
    unsigned long long key = atomicMax(&ws.rest_key[b], 0ull);
    if (key == 0ull) key = atomicMax(&ws.p_key[b], 0ull);
    next = key == 0ull ? 0 : (long long)(0xffffffffu - (unsigned)(key & 0xffffffffull));
  }
  for (int j = threadIdx.x; j < T1; j += kThreads)
    p.out_tokens[(long long)b * T1 + j] = j < k ? p.tokens[b * p.tok_s[0] + j * p.tok_s[1]] : j == k ? next : -1ll;
  if (threadIdx.x == 0) p.accepted[b] = k;
}

template <typename T>
cudaError_t verify(const VerifyParams &p, cudaStream_t stream) {
  const VerifyLayout l = verify_layout(p.drafts, p.vocab);
  const int rows = p.draft.data != nullptr ? (int)l.rows : p.drafts + 1;
  verify_stats_kernel<T><<<dim3(l.chunks, rows, p.batch), kThreads, 0, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  verify_pick_kernel<T><<<dim3(l.chunks, p.batch), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

size_t verify_workspace_bytes(long long batch, long long drafts, long long vocab) {
  const VerifyLayout l = verify_layout(drafts, vocab);
  return (size_t)(align16(batch * 20) + batch * l.rows * l.chunks * 16);
}

cudaError_t launch_verify(const VerifyParams &p, int sms, cudaStream_t stream) {
  (void)sms;
  if (p.batch == 0) return cudaSuccess;
  if (p.dtype == 0) return verify<float>(p, stream);
  if (p.dtype == 1) return verify<__nv_bfloat16>(p, stream);
  return verify<__half>(p, stream);
}

}  // namespace rtk
