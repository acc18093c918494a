// Verification of drafted tokens (speculative decoding) from given random numbers.
//
// Draft t of a sequence is kept while u_t * q_t(x_t) < p_t(x_t); the token after
// the a kept ones is drawn from the positive part of p_a - q_a, or from p_a
// where every draft was kept.  Probabilities enter as whole numbers of 2^-38, so
// sums are exact, the drawn token does not depend on the order in which the
// vocabulary is summed, and a call gives the same token on every GPU.  (2^-38 is
// 3.6e-12: what a vocabulary of 128 k entries loses to the rounding is below
// 5e-7 of the whole, the size of one fp32 rounding of a softmax sum.)
//
// A cluster of CTAs shares one sequence: each finds the number of kept drafts,
// sums its share of the vocabulary (a contiguous share per warp, so that the
// order of tokens is the order of warps) and sends the sum to the others; the
// warp whose share holds the drawn place reads it once more.  One row of p and,
// after a rejection, one of q is all that is read.
#include "wal_kv8.cuh"

#include <cooperative_groups.h>

namespace {

namespace cg = cooperative_groups;
using namespace wal_kv8;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr unsigned long long kOne = 1ull << 38;

struct VerifyParams {
  const float* p;  // [B][T + 1][V]
  long long p_seq, p_row;
  const float* q;  // [B][T][V] or null
  long long q_seq, q_row;
  const int* drafts;
  long long ld_drafts;
  const int* draft_lens;
  const float* u;
  long long ld_u;
  int T, V;
  int* accepted;
  int* tokens;
  long long ld_tokens;
};

__device__ __forceinline__ unsigned long long units(float x) {
  x = fminf(fmaxf(x, 0.f), 1.f);  // a NaN becomes 0
  return (unsigned long long)__float2ll_rn(x * (float)kOne);
}
__device__ __forceinline__ unsigned long long uniform24(float u) {
  u = fminf(fmaxf(u, 0.f), 0.99999994f);
  return (unsigned long long)(u * 16777216.f);
}

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// Weight of token v: the positive part of p - q, of p less the refused draft `out`, or p.
__device__ __forceinline__ unsigned long long weight(float p, float q, bool has_q, bool refused) {
  const unsigned long long pv = units(p), qv = has_q ? units(q) : refused ? kOne : 0ull;
  return pv > qv ? pv - qv : 0ull;
}

__global__ void __launch_bounds__(kThreads) verify_kernel(const __grid_constant__ VerifyParams p) {
  constexpr int U = 8;  // loads in flight per lane and row
  __shared__ int s_a;
  __shared__ unsigned long long warps[kWarps];
  __shared__ unsigned long long ctas[2][kMaxCluster];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), ncta = (int)cl.num_blocks();
  const int b = blockIdx.x / ncta, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  chain();
  const int* x = p.drafts + b * p.ld_drafts;
  const int len = p.draft_lens ? min(max(p.draft_lens[b], 0), p.T) : p.T;
  const unsigned long long place = uniform24(p.u[b * p.ld_u + p.T]);
  if (tid == 0) s_a = len;
  __syncthreads();
  for (int t = tid; t < len; t += kThreads) {
    const int xt = x[t];
    bool ok = (unsigned)xt < (unsigned)p.V;
    if (ok) {
      const float pv = p.p[b * p.p_seq + t * p.p_row + xt], qv = p.q ? p.q[b * p.q_seq + t * p.q_row + xt] : 1.f;
      ok = uniform24(p.u[b * p.ld_u + t]) * units(qv) < units(pv) << 24;
    }
    if (!ok) atomicMin(&s_a, t);
  }
  __syncthreads();
  const int a = s_a;
  const float* pr = p.p + b * p.p_seq + a * p.p_row;
  const float* qr = p.q && a < len ? p.q + b * p.q_seq + a * p.q_row : nullptr;
  int out = a < len && !p.q ? x[a] : -1;  // a refused draft without probabilities
  if (rank == 0)
    for (int t = tid; t <= p.T; t += kThreads)
      if (t != a) p.tokens[b * p.ld_tokens + t] = t < a ? x[t] : -1;
  if (rank == 0 && tid == 0) p.accepted[b] = a;
  const int per = (p.V + ncta * kWarps - 1) / (ncta * kWarps), w = rank * kWarps + warp;
  const int v0 = min(w * per, p.V), v1 = min(v0 + per, p.V);
  for (int pass = 0; pass < 2; ++pass) {  // the second one draws from p itself where the residual is empty
    unsigned long long sum = 0;
    for (int v = v0 + lane; v < v1; v += 32 * U) {
      float pv[U], qv[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const bool in = v + 32 * i < v1;
        pv[i] = in ? __ldg(pr + v + 32 * i) : 0.f;
        qv[i] = in && qr ? __ldg(qr + v + 32 * i) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < U; ++i) sum += weight(pv[i], qv[i], qr, v + 32 * i == out);
    }
    sum = warp_sum(sum);
    if (lane == 0) warps[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      const unsigned long long mine = warp_sum(warps[lane]);
      if (lane < ncta) cl.map_shared_rank(&ctas[pass][0], lane)[rank] = mine;
    }
    cl.sync();
    unsigned long long before = 0, total = 0;
    for (int i = 0; i < ncta; ++i) {
      if (i < rank) before += ctas[pass][i];
      total += ctas[pass][i];
    }
    if (total == 0) {  // nothing is left: p itself, or no token
      if (pass == 1 && rank == 0 && tid == 0) p.tokens[b * p.ld_tokens + a] = -1;
      qr = nullptr;
      out = -1;
      __syncthreads();
      continue;
    }
    const unsigned long long r = (((total >> 32) * place) << 8) + (((total & 0xffffffffull) * place) >> 24);
    for (int i = 0; i < warp; ++i) before += warps[i];
    if (before <= r && r < before + sum) {
      for (int v = v0; v < v1; v += 32) {
        unsigned long long inc = 0;
        if (v + lane < v1) inc = weight(__ldg(pr + v + lane), qr ? __ldg(qr + v + lane) : 0.f, qr, v + lane == out);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += y;
        }
        const unsigned over = __ballot_sync(0xffffffffu, before + inc > r);
        if (over) {
          if (lane == 0) p.tokens[b * p.ld_tokens + a] = v + __ffs(over) - 1;
          break;
        }
        before += __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    break;
  }
}

// CTAs of a cluster: many for few sequences, which leave SMs idle; a batch that
// fills the GPU pays for each CTA's start and barriers.  V = 128256 on B200: 64
// sequences 40.8 us with 8, 33.7 with 4, 40.5 with 2.
int cluster_of(int64_t B) { return B * kMaxCluster <= 2 * sm_count() ? kMaxCluster : 4; }

}  // namespace

extern "C" int wal_verify_drafts(const float* target, int64_t target_seq, int64_t target_row, const float* draft,
                                 int64_t draft_seq, int64_t draft_row, const int32_t* drafts, int64_t ld_drafts,
                                 const int32_t* draft_lens, const float* uniforms, int64_t ld_uniforms, int64_t B,
                                 int64_t T, int64_t V, int32_t* accepted, int32_t* tokens, int64_t ld_tokens,
                                 void* stream) {
  if (!target || !uniforms || !accepted || !tokens || (T > 0 && !drafts)) return WAL_ERR_INVALID_ARGUMENT;
  if (B <= 0 || B > 65535 || T < 0 || T > 4096 || V <= 0 || V > (1 << 22)) return WAL_ERR_SHAPE;
  if (target_row < V || target_seq < 0 || (draft && (draft_row < V || draft_seq < 0))) return WAL_ERR_SHAPE;
  if (ld_drafts < T || ld_uniforms < T + 1 || ld_tokens < T + 1) return WAL_ERR_SHAPE;
  VerifyParams p = {target, target_seq, target_row, draft, draft_seq, draft_row, drafts, ld_drafts, draft_lens, uniforms,
                    ld_uniforms, (int)T, (int)V, accepted, tokens, ld_tokens};
  const int cluster = cluster_of(B);
  return launch_chain(verify_kernel, dim3((unsigned)(B * cluster)), kThreads, 0, static_cast<cudaStream_t>(stream), p, cluster);
}
