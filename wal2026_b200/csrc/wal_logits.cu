// Rules on logits (penalties for repeated tokens, biases, masks, temperature) and
// their softmax, for the T rows of each sequence that a step makes.
//
// A cluster of CTAs takes one row: each keeps its share of the vocabulary in
// shared memory as fp32, so logits are read and outputs written once.  The
// text's tokens are counted in the same place before the logits arrive: every CTA
// reads the text and adds up what falls into its share.  The CTAs then
// exchange (maximum, sum) through distributed shared memory, once: entries are
// held as exp(x - the CTA's maximum), and the factor to the cluster's maximum and
// sum is one number per CTA.
//
// Numerics: everything is fp32, in the order of the definition; x / repetition,
// x / temperature and exp are the full-precision ones.
#include "wal_kv8.cuh"

#include <cuda_fp16.h>

#include <cooperative_groups.h>

namespace {

namespace cg = cooperative_groups;
using wal_kv8::kMaxDevices;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kMaxShare = 49152;  // entries of a CTA: 192 KB
constexpr int kMaxBias = 1024;

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

constexpr unsigned kPrompt = 0x80000000u;  // a token of the prompt; the other bits count generated ones

__device__ __forceinline__ float penalise(float x, unsigned c, float rep, float freq, float pres) {
  if (c == 0u) return x;
  x = x > 0.f ? x / rep : x * rep;
  const unsigned made = c & ~kPrompt;
  if (made) x = x - freq * (float)made - pres;
  return x;
}

// (value, index) of the larger value, the lower index among equals
__device__ __forceinline__ void better(float& v, int& i, float v2, int i2) {
  if (v2 > v || (v2 == v && i2 < i)) {
    v = v2;
    i = i2;
  }
}

// VEC: rows of logits and outputs are aligned for four entries.
template <int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) logit_rules_kernel(const __grid_constant__ RulesParams p) {
  extern __shared__ __align__(16) float xs[];  // this CTA's entries; counts first
  __shared__ int ids[kMaxBias];
  __shared__ float adds[kMaxBias];
  __shared__ float wv[kWarps], wsum[kWarps];
  __shared__ int wi[kWarps];
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
  float* out = p.out + b * p.out_seq + t * p.out_row + v0;
  const bool idle = p.r.new_lens && t >= p.r.new_lens[b];
  const bool counted = p.r.repetition || p.r.presence || p.r.frequency;
  const float rep = p.r.repetition ? p.r.repetition[b] : 1.f, pres = p.r.presence ? p.r.presence[b] : 0.f;
  const float freq = p.r.frequency ? p.r.frequency[b] : 0.f, temp = p.r.temperature ? p.r.temperature[b] : 1.f;
  const bool greedy = !(temp > 0.f);

  if (counted && !idle) {
    unsigned* cnt = reinterpret_cast<unsigned*>(xs);
    for (int i = tid; i < (n + 3) / 4; i += kThreads) reinterpret_cast<uint4*>(cnt)[i] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    const int* text = p.r.text + b * p.r.ld_text;
    const long long upto = min((long long)max(p.r.lens[b], -1 - t) + t + 1, (long long)p.r.text_len);
    const int prompt = p.r.prompt_lens ? p.r.prompt_lens[b] : 0;
    for (long long j = tid; j < upto; j += kThreads) {
      const unsigned at = (unsigned)text[j] - (unsigned)v0;
      if (at < (unsigned)n) {
        if (j < prompt) atomicOr(cnt + at, kPrompt);
        else atomicAdd(cnt + at, 1u);
      }
    }
    __syncthreads();
  }
  // x, penalised and masked
  if (!idle) {
    const long long base = b * p.ld_seq + t * p.ld_row + v0;
    const int* mask = p.r.mask ? p.r.mask + b * p.r.mask_seq + t * p.r.mask_row : nullptr;
    for (int i = 4 * tid; i < n; i += 4 * kThreads) {
      float x[4];
      if (VEC) {
        const float4 f = load4<DT>(p.logits, base + i);
        x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = i + e < n ? load1<DT>(p.logits, base + i + e) : -INFINITY;
      }
      const unsigned bits = mask ? (unsigned)__ldg(mask + ((v0 + i) >> 5)) >> ((v0 + i) & 31) : 15u;
      if (counted) {
        const uint4 c = *reinterpret_cast<const uint4*>(xs + i);
        x[0] = penalise(x[0], c.x, rep, freq, pres);
        x[1] = penalise(x[1], c.y, rep, freq, pres);
        x[2] = penalise(x[2], c.z, rep, freq, pres);
        x[3] = penalise(x[3], c.w, rep, freq, pres);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!((bits >> e) & 1) || !(x[e] == x[e])) x[e] = -INFINITY;
      *reinterpret_cast<float4*>(xs + i) = make_float4(x[0], x[1], x[2], x[3]);
    }
  }
  if (p.r.num_bias > 0 && !idle) {
    const int nb = (int)p.r.num_bias;
    for (int i = tid; i < nb; i += kThreads) {
      ids[i] = p.r.bias_ids[b * p.r.num_bias + i];
      adds[i] = p.r.bias[b * p.r.num_bias + i];
    }
    __syncthreads();
    for (int i = tid; i < nb; i += kThreads) {
      const unsigned at = (unsigned)ids[i] - (unsigned)v0;
      if (at >= (unsigned)n) continue;
      bool first = true;
      for (int j = 0; j < i; ++j) first &= ids[j] != ids[i];
      if (!first) continue;  // the first of equal ones adds them all, in order
      float sum = adds[i];
      for (int j = i + 1; j < nb; ++j)
        if (ids[j] == ids[i]) sum += adds[j];
      const float x = xs[at];
      if (x != -INFINITY) xs[at] = x + sum == x + sum ? x + sum : -INFINITY;
    }
  }
  __syncthreads();

  // this CTA's largest, and its sum relative to it
  float top = -INFINITY;
  int where = 0x7fffffff;
  if (!idle) {
    for (int i = tid; i < n; i += kThreads) {
      float x = xs[i];
      if (!greedy && p.r.temperature) {
        x = x / temp;
        if (!(x == x)) x = -INFINITY;
        xs[i] = x;
      }
      better(top, where, x, v0 + i);
    }
  }
  if (!p.softmax) {
    for (int i = tid; i < n; i += kThreads) out[i] = idle ? 0.f : xs[i];
    asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
    return;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) better(top, where, __shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, where, o));
  if (lane == 0) wv[warp] = top, wi[warp] = where;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) better(top, where, wv[w], wi[w]);
  float sum = 0.f;
  if (!idle && !greedy && top > -INFINITY) {
    for (int i = tid; i < n; i += kThreads) {
      const float x = xs[i], e = x == top ? 1.f : expf(x - top);
      xs[i] = e;
      sum += e;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) wsum[warp] = sum;
  __syncthreads();
  asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
  if (tid < ncta) {
    float s = 0.f;
    for (int w = 0; w < kWarps; ++w) s += wsum[w];
    *cl.map_shared_rank(&cmax[rank], tid) = top;
    *cl.map_shared_rank(&csum[rank], tid) = s;
    *cl.map_shared_rank(&cidx[rank], tid) = where;
  }
  cl.sync();
  float all = -INFINITY;
  int best = 0x7fffffff;
  for (int c = 0; c < ncta; ++c) better(all, best, cmax[c], cidx[c]);
  float total = 0.f;
  for (int c = 0; c < ncta; ++c)
    if (cmax[c] > -INFINITY) total += csum[c] * (cmax[c] == all ? 1.f : expf(cmax[c] - all));
  const float factor = idle || greedy || !(top > -INFINITY) ? 0.f : (top == all ? 1.f : expf(top - all)) / total;
  const int one = !idle && greedy && all > -INFINITY ? best - v0 : -1;
  for (int i = 4 * tid; i < n; i += 4 * kThreads) {
    float4 e = factor == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(xs + i);
    e.x = i == one ? 1.f : e.x * factor;
    e.y = i + 1 == one ? 1.f : e.y * factor;
    e.z = i + 2 == one ? 1.f : e.z * factor;
    e.w = i + 3 == one ? 1.f : e.w * factor;
    if (VEC) {
      *reinterpret_cast<float4*>(out + i) = e;
    } else {
      out[i] = e.x;
      if (i + 1 < n) out[i + 1] = e.y;
      if (i + 2 < n) out[i + 2] = e.z;
      if (i + 3 < n) out[i + 3] = e.w;
    }
  }
}

template <int DT, bool VEC>
int launch(const RulesParams& p, int cluster, cudaStream_t st) {
  auto kern = logit_rules_kernel<DT, VEC>;
  static std::atomic<uint64_t> allowed{0};  // devices where the kernel may use its shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return WAL_ERR_CUDA;
  if (!(allowed.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxShare * 4) != cudaSuccess) return WAL_ERR_CUDA;
    allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  return wal_kv8::launch_chain(kern, dim3((unsigned)(p.B * p.T * cluster)), kThreads, p.share * 4, st, p, cluster);
}

template <int DT>
int launch_type(const RulesParams& p, bool vec, int cluster, cudaStream_t st) {
  return vec ? launch<DT, true>(p, cluster, st) : launch<DT, false>(p, cluster, st);
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
  if (B <= 0 || T <= 0 || V <= 0 || V > (int64_t)kMaxShare * kMaxCluster || B >= (1 << 27) || T >= (1 << 27) || B * T >= (1 << 27))
    return WAL_ERR_SHAPE;
  if (ld_seq < 0 || ld_row < V || out_row < V || out_seq < 0 || (B > 1 && out_seq < (T - 1) * out_row + V)) return WAL_ERR_SHAPE;
  if (r.text && (r.text_len < 0 || r.ld_text < r.text_len || r.text_len > 0x7fffffff)) return WAL_ERR_SHAPE;
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
