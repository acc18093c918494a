// Rules on logits (penalties for repeated tokens, biases, masks, temperature) and
// their softmax, for the T rows of each sequence that a step makes.
//
// A cluster of CTAs takes one row and each thread some groups of four entries of
// it, in registers, so logits are read and outputs written once.  What the rules
// know of an entry is a word in shared memory: how often the text has it, whether
// the prompt does, and which bias it has; most words are zero and cost a test per
// group.  Every CTA reads the text and counts what falls into its share while its
// logits are on their way.  The CTAs exchange (maximum, sum) through distributed
// shared memory once: entries are held as exp(x - the CTA's maximum), and the
// factor to the cluster's maximum and sum is one number per CTA.
//
// Numerics: fp32 in the order of the definition.  The temperature goes into the
// exponent: exp(x / t - m / t) = exp2(x k - m k), k = log2(e) / t, in one fused
// multiply-add, off by 2^-24 of the exponent and a rounding of m k that all of the CTA's
// entries share.  Temperatures outside [2^-40, 2^40] and maxima near fp32's ends
// divide and subtract instead.
#include "wal_kv8.cuh"

#include <cuda_fp16.h>

#include <cooperative_groups.h>

namespace {

namespace cg = cooperative_groups;
using wal_kv8::kMaxDevices;

constexpr int kMaxCluster = 8;
constexpr int kMaxVocab = 393216;
constexpr int kMaxBias = 1024;
constexpr int kMaxText = (1 << 20) - 1;

struct RulesParams {
  wal_logit_rules r;
  const void* logits;
  long long ld_seq, ld_row;
  float* out;
  long long out_seq, out_row;
  int B, T, V, share;  // entries per CTA, a multiple of 4
  int softmax;
};

template <int DT>
__device__ __forceinline__ float load1(const void* p, long long i) {
  if (DT == WAL_F32) return __ldg(static_cast<const float*>(p) + i);
  const unsigned short u = __ldg(static_cast<const unsigned short*>(p) + i);
  return DT == WAL_F16 ? __half2float(__ushort_as_half(u)) : __uint_as_float((uint32_t)u << 16);
}

template <int DT>
__device__ __forceinline__ float4 load4(const void* p, long long i) {
  if (DT == WAL_F32) return __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + i));
  const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const unsigned short*>(p) + i));
  if (DT == WAL_BF16) return make_float4(wal_kv8::bf16_lo(w.x), wal_kv8::bf16_hi(w.x), wal_kv8::bf16_lo(w.y), wal_kv8::bf16_hi(w.y));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

// What the rules know of an entry: bits 0 to 19 times generated, bit 20 in the prompt, from bit 21 its bias (from 1).
constexpr unsigned kCount = (1u << 20) - 1, kPrompt = 1u << 20;
constexpr int kBiasBit = 21;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// x, and -inf for a NaN (of a maximum with -inf the compiler would keep the other side)
__device__ __forceinline__ float number(float x) {
  float y;
  asm("max.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(-INFINITY));
  return y;
}

// (value, index) of the larger value, the lower index among equals
__device__ __forceinline__ void better(float& v, int& i, float v2, int i2) {
  if (v2 > v || (v2 == v && i2 < i)) {
    v = v2;
    i = i2;
  }
}

// NT threads with K groups of four entries each.  VEC: rows of logits and outputs are aligned for groups.
template <int DT, bool VEC, int K, int NT>
__global__ void __launch_bounds__(NT, NT == 512 ? 2 : 1) logit_rules_kernel(const __grid_constant__ RulesParams p) {
  constexpr int W = NT / 32;
  extern __shared__ __align__(16) unsigned words[];  // of this CTA's entries, where the rules ask for them
  __shared__ int ids[kMaxBias];
  __shared__ float adds[kMaxBias];
  __shared__ float wv[W], wsum[W];
  __shared__ int wi[W];
  __shared__ float cmax[kMaxCluster], csum[kMaxCluster];
  __shared__ int cidx[kMaxCluster];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), ncta = (int)cl.num_blocks();
  const long long row = blockIdx.x / ncta;
  const int b = (int)(row / p.T), t = (int)(row % p.T);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  wal_kv8::chain();
  // a CTA's shared memory may be written by the others once it has started
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");
  const int v0 = min(rank * p.share, p.V), n = min(p.share, p.V - v0);
  float* const out = p.out + b * p.out_seq + t * p.out_row + v0;
  const bool idle = p.r.new_lens && t >= p.r.new_lens[b];
  auto write = [&](int i, const float (&v)[4]) {
    if (VEC) {
      if (i < n) __stcs(reinterpret_cast<float4*>(out + i), make_float4(v[0], v[1], v[2], v[3]));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < n) out[i + e] = v[e];
    }
  };
  if (idle) {
    const float none[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < K; ++k) write(4 * (tid + NT * k), none);
    asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
    return;  // all CTAs of the row do
  }
  float x[K][4];
  const long long base = b * p.ld_seq + t * p.ld_row + v0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = 4 * (tid + NT * k);
    if (VEC) {
      const float4 f = i < n ? load4<DT>(p.logits, base + i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      x[k][0] = f.x, x[k][1] = f.y, x[k][2] = f.z, x[k][3] = f.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[k][e] = i + e < n ? load1<DT>(p.logits, base + i + e) : -INFINITY;
    }
  }
  const bool counted = p.r.repetition || p.r.presence || p.r.frequency;
  const int nb = (int)p.r.num_bias;
  if (counted || nb) {
    for (int i = tid; i < (n + 3) / 4; i += NT) reinterpret_cast<uint4*>(words)[i] = make_uint4(0u, 0u, 0u, 0u);
    for (int i = tid; i < nb; i += NT) {
      ids[i] = p.r.bias_ids[(long long)b * nb + i];
      adds[i] = p.r.bias[(long long)b * nb + i];
    }
    __syncthreads();
    if (counted) {
      const int* text = p.r.text + b * p.r.ld_text;
      const int upto = (int)min((long long)max(p.r.lens[b], -1 - t) + t + 1, (long long)p.r.text_len);
      const int prompt = p.r.prompt_lens ? p.r.prompt_lens[b] : 0;
#pragma unroll 4
      for (int j = tid; j < upto; j += NT) {
        const unsigned at = (unsigned)text[j] - (unsigned)v0;
        if (at < (unsigned)n) {
          if (j < prompt) atomicOr(words + at, kPrompt);
          else atomicAdd(words + at, 1u);
        }
      }
    }
    float sum = 0.f;
    for (int i = tid; i < nb; i += NT) {
      const unsigned at = (unsigned)ids[i] - (unsigned)v0;
      if (at >= (unsigned)n) continue;
      bool first = true;
      for (int j = 0; j < i && first; ++j) first = ids[j] != ids[i];
      if (!first) continue;  // the first of equal ones adds them all, in order
      sum = adds[i];
      for (int j = i + 1; j < nb; ++j)
        if (ids[j] == ids[i]) sum += adds[j];
      atomicOr(words + at, (unsigned)(i + 1) << kBiasBit);
      if (sum != adds[i]) adds[i] = sum;  // no other thread reads the first one's
    }
    __syncthreads();
  }
  const float rep = p.r.repetition ? p.r.repetition[b] : 1.f, pres = p.r.presence ? p.r.presence[b] : 0.f;
  const float freq = p.r.frequency ? p.r.frequency[b] : 0.f, temp = p.r.temperature ? p.r.temperature[b] : 1.f;
  const bool greedy = !(temp > 0.f);
  const int* const mask = p.r.mask ? p.r.mask + b * p.r.mask_seq + t * p.r.mask_row : nullptr;
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = 4 * (tid + NT * k);
    if ((counted || nb) && i < n) {
      const uint4 c = *reinterpret_cast<const uint4*>(words + i);
      if (c.x | c.y | c.z | c.w) {
        const unsigned w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (w[e] & (kCount | kPrompt)) {
            x[k][e] = x[k][e] > 0.f ? x[k][e] / rep : x[k][e] * rep;
            if (w[e] & kCount) x[k][e] = x[k][e] - freq * (float)(w[e] & kCount) - pres;
          }
          if (w[e] >> kBiasBit) x[k][e] += adds[(w[e] >> kBiasBit) - 1];
        }
      }
    }
    if (mask) {
      const unsigned bits = i < n ? (unsigned)__ldg(mask + ((v0 + i) >> 5)) >> ((v0 + i) & 31) : 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[k][e] = (bits >> e) & 1 ? x[k][e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[k][e] = number(x[k][e]);
      top = fmaxf(top, x[k][e]);
    }
  }
  if (!p.softmax) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!greedy && p.r.temperature)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k][e] = number(x[k][e] / temp);
      write(4 * (tid + NT * k), x[k]);
    }
    asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
    return;
  }
  // this CTA's largest, and its sum relative to it
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) wv[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) top = fmaxf(top, wv[w]);
  const float scale = 1.4426950408889634f / temp, off = -top * scale;
  const bool usual = temp >= 9.0949470177292824e-13f && temp <= 1.099511627776e12f && fabsf(off) < 1e30f;
  float sum = 0.f, ref = top;  // ref: what this CTA's entries are relative to, divided by the temperature
  int where = 0x7fffffff;
  if (greedy) {
#pragma unroll
    for (int k = K - 1; k >= 0; --k)
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (x[k][e] == top) where = v0 + 4 * (tid + NT * k) + e;
  } else if (usual) {
    ref = top / temp;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[k][e] = ex2(fmaf(x[k][e], scale, off));
        sum += x[k][e];
      }
  } else {
    ref = number(top / temp);
    // a temperature can make the largest infinite, or a NaN of an infinite one: then what is equal to it shares
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y = number(x[k][e] / temp);
        x[k][e] = y == -INFINITY ? 0.f : y == ref ? 1.f : expf(y - ref);
        sum += x[k][e];
      }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    where = min(where, __shfl_xor_sync(0xffffffffu, where, o));
  }
  if (lane == 0) wsum[warp] = sum, wi[warp] = where;
  __syncthreads();
  asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
  if (tid < ncta) {
    float s = 0.f;
    int first = 0x7fffffff;
    for (int w = 0; w < W; ++w) {
      s += wsum[w];
      first = min(first, wi[w]);
    }
    *cl.map_shared_rank(&cmax[rank], tid) = ref;
    *cl.map_shared_rank(&csum[rank], tid) = s;
    *cl.map_shared_rank(&cidx[rank], tid) = first;
  }
  cl.sync();
  float all = -INFINITY, total = 0.f;
  int best = 0x7fffffff;
  for (int c = 0; c < ncta; ++c) better(all, best, cmax[c], cidx[c]);
  for (int c = 0; c < ncta; ++c)
    if (cmax[c] > -INFINITY) total += csum[c] * (cmax[c] == all ? 1.f : expf(cmax[c] - all));
  const float factor = greedy || !(ref > -INFINITY) ? 0.f : (ref == all ? 1.f : expf(ref - all)) / total;
  const int one = greedy && all > -INFINITY ? best - v0 : -1;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = 4 * (tid + NT * k);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[k][e] = factor == 0.f ? (i + e == one ? 1.f : 0.f) : x[k][e] * factor;
    write(i, x[k]);
  }
}

template <int DT, bool VEC, int K, int NT>
int launch(const RulesParams& p, int cluster, cudaStream_t st) {
  auto kern = logit_rules_kernel<DT, VEC, K, NT>;
  const bool words = p.r.repetition || p.r.presence || p.r.frequency || p.r.num_bias;
  static std::atomic<uint64_t> allowed{0};  // devices where the kernel may use its shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return WAL_ERR_CUDA;
  if (!(allowed.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * NT * K * 4) != cudaSuccess) return WAL_ERR_CUDA;
    allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  return wal_kv8::launch_chain(kern, dim3((unsigned)(p.B * p.T * cluster)), NT, words ? p.share * 4 : 0, st, p, cluster);
}

// A thread holds as few groups as its CTA's share needs; shares beyond 16384 take twice the threads.
template <int DT, bool VEC>
int launch_share(const RulesParams& p, int cluster, cudaStream_t st) {
  if (p.share <= 2048) return launch<DT, VEC, 1, 512>(p, cluster, st);
  if (p.share <= 8192) return launch<DT, VEC, 4, 512>(p, cluster, st);
  if (p.share <= 16384) return launch<DT, VEC, 8, 512>(p, cluster, st);
  return launch<DT, VEC, 12, 1024>(p, cluster, st);
}

template <int DT>
int launch_type(const RulesParams& p, bool vec, int cluster, cudaStream_t st) {
  return vec ? launch_share<DT, true>(p, cluster, st) : launch_share<DT, false>(p, cluster, st);
}

}  // namespace

extern "C" {

int wal_logit_rules_apply(const wal_logit_rules* rules, const void* logits, int dtype, int64_t ld_seq, int64_t ld_row, int64_t B,
                          int64_t T, int64_t V, float* out, int64_t out_seq, int64_t out_row, int softmax, void* stream) {
  if (!rules || !logits || !out) return WAL_ERR_INVALID_ARGUMENT;
  const wal_logit_rules& r = *rules;
  if ((r.repetition || r.presence || r.frequency) && (!r.lens || (!r.text && r.text_len))) return WAL_ERR_INVALID_ARGUMENT;
  if (!r.bias_ids != !r.bias || (!r.bias_ids && r.num_bias)) return WAL_ERR_INVALID_ARGUMENT;
  if (dtype != WAL_BF16 && dtype != WAL_F32 && dtype != WAL_F16) return WAL_ERR_UNSUPPORTED;
  if (B <= 0 || T <= 0 || V <= 0 || V > kMaxVocab || B >= (1 << 27) || T >= (1 << 27) || B * T >= (1 << 27))
    return WAL_ERR_SHAPE;
  if (ld_seq < 0 || ld_row < V || out_row < V || out_seq < 0 || (B > 1 && out_seq < (T - 1) * out_row + V)) return WAL_ERR_SHAPE;
  if (r.text && (r.text_len < 0 || r.ld_text < r.text_len || r.text_len > kMaxText)) return WAL_ERR_SHAPE;
  if (r.num_bias < 0 || r.num_bias > kMaxBias || r.mask_seq < 0 || r.mask_row < 0) return WAL_ERR_SHAPE;
  const int size = dtype == WAL_F32 ? 4 : 2;
  if (((uintptr_t)logits & (size - 1)) || ((uintptr_t)out & 3)) return WAL_ERR_ALIGNMENT;
  RulesParams p = {};
  p.r = r;
  p.logits = logits;
  p.ld_seq = ld_seq;
  p.ld_row = ld_row;
  p.out = out;
  p.out_seq = out_seq;
  p.out_row = out_row;
  p.B = (int)B;
  p.T = (int)T;
  p.V = (int)V;
  p.softmax = softmax;
  int cluster = 1;
  while (cluster < kMaxCluster && V > cluster * 2048) cluster *= 2;
  p.share = (int)(((V + cluster - 1) / cluster + 31) & ~31);
  const bool vec = V % 4 == 0 && ld_row % 4 == 0 && ld_seq % 4 == 0 && out_row % 4 == 0 && out_seq % 4 == 0 &&
                   !((uintptr_t)logits & (4 * size - 1)) && !((uintptr_t)out & 15);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == WAL_BF16) return launch_type<WAL_BF16>(p, vec, cluster, st);
  if (dtype == WAL_F16) return launch_type<WAL_F16>(p, vec, cluster, st);
  return launch_type<WAL_F32>(p, vec, cluster, st);
}

}  // extern "C"
