// Verification of drafted tokens (speculative decoding) from given random numbers.
//
// Draft t of a sequence is kept while u_t * q_t(x_t) < p_t(x_t); the token after
// the a kept ones is drawn from the positive part of p_a - q_a, or from p_a
// where every draft was kept.  Probabilities enter as whole numbers of 2^-38, so
// sums are exact, the drawn token does not depend on the order in which the
// vocabulary is summed, and a call gives the same token on every GPU.  (2^-38 is
// 3.6e-12: what a vocabulary of 128 k entries loses to the rounding is below
// 5e-7 of the whole, the size of one fp32 rounding of a softmax sum.)
#include "../../include/wal_rvq.h"

#include <cuda_runtime.h>
#include <stdint.h>

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
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

__global__ void __launch_bounds__(kThreads) verify_kernel(const __grid_constant__ VerifyParams p) {
  __shared__ int s_a, s_token;
  __shared__ unsigned long long sums[kWarps];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int* x = p.drafts + b * p.ld_drafts;
  const int len = p.draft_lens ? min(max(p.draft_lens[b], 0), p.T) : p.T;
  if (tid == 0) s_a = len, s_token = -1;
  __syncthreads();
  for (int t = tid; t < len; t += kThreads) {
    const int xt = x[t];
    bool ok = (unsigned)xt < (unsigned)p.V;
    if (ok) {
      const unsigned long long px = units(p.p[b * p.p_seq + t * p.p_row + xt]);
      const unsigned long long qx = p.q ? units(p.q[b * p.q_seq + t * p.q_row + xt]) : kOne;
      ok = uniform24(p.u[b * p.ld_u + t]) * qx < px << 24;
    }
    if (!ok) atomicMin(&s_a, t);
  }
  __syncthreads();
  const int a = s_a;
  const float* pr = p.p + b * p.p_seq + a * p.p_row;
  const float* qr = p.q && a < len ? p.q + b * p.q_seq + a * p.q_row : nullptr;
  int out = a < len && !p.q ? x[a] : -1;  // a rejected draft without probabilities
  const int per = (p.V + kThreads - 1) / kThreads, v0 = min(tid * per, p.V), v1 = min(v0 + per, p.V);
  for (int pass = 0; pass < 2; ++pass) {  // the second one draws from p itself where the residual is empty
    unsigned long long w = 0;
    for (int v = v0; v < v1; ++v) {
      const unsigned long long pv = units(pr[v]), qv = qr ? units(qr[v]) : (v == out ? kOne : 0ull);
      w += pv > qv ? pv - qv : 0ull;
    }
    unsigned long long inc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    unsigned long long before = 0, total = 0;
    for (int i = 0; i < kWarps; ++i) {
      if (i < warp) before += sums[i];
      total += sums[i];
    }
    if (total) {
      const unsigned long long u = uniform24(p.u[b * p.ld_u + p.T]);
      const unsigned long long r = (((total >> 32) * u) << 8) + (((total & 0xffffffffull) * u) >> 24);
      unsigned long long c = before + inc - w;
      if (c <= r && r < c + w) {
        for (int v = v0; v < v1; ++v) {
          const unsigned long long pv = units(pr[v]), qv = qr ? units(qr[v]) : (v == out ? kOne : 0ull);
          c += pv > qv ? pv - qv : 0ull;
          if (c > r) {
            s_token = v;
            break;
          }
        }
      }
      break;
    }
    qr = nullptr;
    out = -1;
    __syncthreads();
  }
  __syncthreads();
  for (int t = tid; t <= p.T; t += kThreads)
    p.tokens[b * p.ld_tokens + t] = t < a ? x[t] : t == a ? s_token : -1;
  if (tid == 0) p.accepted[b] = a;
}

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
  verify_kernel<<<(unsigned)B, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return cudaGetLastError() == cudaSuccess ? WAL_OK : WAL_ERR_CUDA;
}
