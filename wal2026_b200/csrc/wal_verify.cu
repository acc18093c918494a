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
//
// On B200, 128256 tokens: one sequence 6.9 us (1 MB: three dependent loads, the
// sums, a cluster barrier and the second reading of one share), 64 sequences 20.4 us for 66
// MB, 3.2 TB/s: half the time is the same chain before and after the rows stream.
#include "wal_kv8.cuh"

#include <cooperative_groups.h>

namespace {

namespace cg = cooperative_groups;
using namespace wal_kv8;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;

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

// round(2^38 x) of x clamped to [0, 1] (NaN as 0), as hi * 2^23 + lo: adding 2^23
// to 2^15 x rounds it to a whole number, and what is left is exact and takes 23
// bits more in the same way.  The bit patterns of the two sums count from
// kHiBits and kLoBits.  (A conversion to 64-bit integers does the same at a
// fraction of the rate.)
struct Fixed {
  uint32_t hi, lo;
};
constexpr uint32_t kHiBits = 0x4b000000u, kLoBits = 0x4b400000u;  // 2^23, 1.5 * 2^23

__device__ __forceinline__ Fixed fixed(float x) {
  x = __saturatef(x);
  const float t = __fmaf_rn(x, 32768.f, 8388608.f);
  const float rest = __fmaf_rn(x, 32768.f, -__fadd_rn(t, -8388608.f));
  return {__float_as_uint(t), __float_as_uint(__fmaf_rn(rest, 8388608.f, 12582912.f))};
}

__device__ __forceinline__ long long difference(const Fixed& a, uint32_t hi, uint32_t lo) {
  return (long long)(int)(a.hi - hi) * 8388608ll + (int)(a.lo - lo);
}

__device__ __forceinline__ unsigned long long units(float x) { return (unsigned long long)difference(fixed(x), kHiBits, kLoBits); }

__device__ __forceinline__ unsigned long long uniform24(float u) {
  u = fminf(fmaxf(u, 0.f), 0.99999994f);
  return (unsigned long long)(u * 16777216.f);
}

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// hi * 2^23 + lo += P - min(P, Q); parts of 16 weights fit.
__device__ __forceinline__ void add_weight(float p, float q, uint32_t& hi, uint32_t& lo) {
  p = __saturatef(p);
  const Fixed f = fixed(p), g = fixed(fminf(p, __saturatef(q)));
  hi += f.hi - g.hi;
  lo += f.lo - g.lo;
}

// Weight of a token: the positive part of p - q (q = 0 where there is none), nothing for the refused draft.
__device__ __forceinline__ unsigned long long weight(float p, float q, bool refused) {
  const Fixed f = fixed(q);
  const long long w = difference(fixed(p), f.hi, f.lo);
  return w > 0 && !refused ? (unsigned long long)w : 0ull;
}

// Entries v .. v + 3 of a row, zeros from `end` on.  VEC: the rows are 16-byte aligned, v and end multiples of 4.
template <bool VEC>
__device__ __forceinline__ float4 load4(const float* row, int v, int end) {
  if (VEC) return v < end ? __ldg(reinterpret_cast<const float4*>(row + v)) : make_float4(0.f, 0.f, 0.f, 0.f);
  return make_float4(v < end ? __ldg(row + v) : 0.f, v + 1 < end ? __ldg(row + v + 1) : 0.f,
                     v + 2 < end ? __ldg(row + v + 2) : 0.f, v + 3 < end ? __ldg(row + v + 3) : 0.f);
}

// CTAS: per SM
template <bool VEC, int CTAS>
__global__ void __launch_bounds__(kThreads, CTAS) verify_kernel(const __grid_constant__ VerifyParams p) {
  constexpr int U = 4;  // groups of four entries in flight per lane and row
  __shared__ int s_a;
  __shared__ unsigned long long warps[kWarps];
  __shared__ unsigned long long ctas[2][kMaxCluster];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), ncta = (int)cl.num_blocks();
  const int b = blockIdx.x / ncta, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  chain();
  // a CTA's shared memory may be written by the others once it has started
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");
  const int* x = p.drafts + b * p.ld_drafts;
  const int len = p.draft_lens ? min(max(p.draft_lens[b], 0), p.T) : p.T;
  const unsigned long long place = uniform24(p.u[b * p.ld_u + p.T]);
  if (tid == 0) s_a = len;
  __syncthreads();
  for (int t = tid; t < p.T; t += kThreads) {
    const int xt = x[t];
    bool ok = (unsigned)xt < (unsigned)p.V;
    if (ok && t < len) {
      const float pv = p.p[b * p.p_seq + t * p.p_row + xt], qv = p.q ? p.q[b * p.q_seq + t * p.q_row + xt] : 1.f;
      ok = uniform24(p.u[b * p.ld_u + t]) * units(qv) < units(pv) << 24;
    }
    if (!ok && t < len) atomicMin(&s_a, t);
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
  const int per = ((p.V + ncta * kWarps - 1) / (ncta * kWarps) + 3) & ~3, w = rank * kWarps + warp;
  const int v0 = (int)min((long long)w * per, (long long)p.V), v1 = min(v0 + per, p.V);
  for (int pass = 0; pass < 2; ++pass) {  // the second one draws from p itself where the residual is empty
    unsigned long long sum = 0;
    for (int v = v0 + 4 * lane; v < v1; v += 128 * U) {
      float4 pv[U], qv[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        pv[i] = load4<VEC>(pr, v + 128 * i, v1);
        qv[i] = qr ? load4<VEC>(qr, v + 128 * i, v1) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      // the sum of P - min(P, Q), part by part: the smaller of the two in fp32 has the smaller whole number
      uint32_t hi = 0, lo = 0;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int o = out - (v + 128 * i);
        add_weight(pv[i].x, o == 0 ? pv[i].x : qv[i].x, hi, lo);
        add_weight(pv[i].y, o == 1 ? pv[i].y : qv[i].y, hi, lo);
        add_weight(pv[i].z, o == 2 ? pv[i].z : qv[i].z, hi, lo);
        add_weight(pv[i].w, o == 3 ? pv[i].w : qv[i].w, hi, lo);
      }
      sum += (unsigned long long)((long long)(int)hi * 8388608ll + (int)lo);
    }
    sum = warp_sum(sum);
    if (lane == 0) warps[warp] = sum;
    __syncthreads();
    if (pass == 0) asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
    if (warp == 0) {
      const unsigned long long mine = warp_sum(lane < kWarps ? warps[lane] : 0ull);
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
    if (before <= r && r < before + sum) {  // this warp's share holds the place: its weights once more, in order
      for (int v = v0; v < v1; v += 128) {
        const int at = v + 4 * lane, o = out - at;
        const float4 pv = load4<VEC>(pr, at, v1), qv = qr ? load4<VEC>(qr, at, v1) : make_float4(0.f, 0.f, 0.f, 0.f);
        const unsigned long long w0 = weight(pv.x, qv.x, o == 0), w1 = w0 + weight(pv.y, qv.y, o == 1),
                                 w2 = w1 + weight(pv.z, qv.z, o == 2), w3 = w2 + weight(pv.w, qv.w, o == 3);
        unsigned long long inc = w3;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
          const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, x);
          if (lane >= x) inc += y;
        }
        const unsigned over = __ballot_sync(0xffffffffu, before + inc > r);
        if (over) {
          if (lane == __ffs(over) - 1) {
            const unsigned long long c = before + inc - w3;
            p.tokens[b * p.ld_tokens + a] = at + (c + w0 > r ? 0 : c + w1 > r ? 1 : c + w2 > r ? 2 : 3);
          }
          break;
        }
        before += __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    break;
  }
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
  const bool vec = V % 4 == 0 && target_seq % 4 == 0 && target_row % 4 == 0 && ((uintptr_t)target & 15) == 0 &&
                   (!draft || (draft_seq % 4 == 0 && draft_row % 4 == 0 && ((uintptr_t)draft & 15) == 0));
  // Few sequences leave SMs idle: eight CTAs each, one per SM.  A batch pays for
  // each CTA's start and barriers: four each, two per SM.  V = 128256 on B200:
  // one sequence 6.9 us with eight CTAs one per SM, 7.3 two per SM, 9.6 with four; 64
  // sequences 25.1 us with four CTAs one per SM, 20.4 two per SM, 26.0 with eight.
  const bool few = B * kMaxCluster <= sm_count();
  const int cluster = few ? kMaxCluster : 4;
  auto kern = few ? (vec ? verify_kernel<true, 1> : verify_kernel<false, 1>) : (vec ? verify_kernel<true, 2> : verify_kernel<false, 2>);
  return launch_chain(kern, dim3((unsigned)(B * cluster)), kThreads, 0, static_cast<cudaStream_t>(stream), p, cluster);
}
