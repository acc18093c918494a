// Rules on logits (penalties for repeated tokens, biases, masks, temperature) and
// their softmax, for the T rows of each sequence that a step makes.
//
// A cluster of CTAs takes one row, dealt out in blocks of 128 entries (frequent
// tokens have neighbouring numbers), and each thread some groups of four entries, in registers, so logits are read and outputs written once.  What the rules
// know of an entry is a word in shared memory: how often the text has it, whether
// the prompt does, and which bias it has; most words are zero and cost a test per
// group.  Every CTA reads the text and counts what falls into its share while its
// logits are on their way.  The CTAs exchange (maximum, sum) through distributed
// shared memory once: entries are held as exp((x - the CTA's maximum) / t), and the
// factor to the cluster's maximum and sum is one number per CTA.  Clusters that fill
// the GPU take the rows in order: the T rows of a sequence need one count of the
// text and then a token more each, and the next row's logits are asked into L2
// while this one is worked on.
//
// Numerics: fp32 in the order of the definition, with one change: of exp(x / t - m / t) the
// difference is taken before the division, exp2((x - m) * k), k = log2(e) / t, so that an
// exponent is off by 4 * 2^-24 of itself however far from zero the logits lie.  Maxima
// are exchanged as they are, undivided: every CTA's entries stand relative to a number that
// all know exactly.  (The fused exp2(x k - round(m k)), with each CTA's maximum divided
// anew for the exchange, was off by 2^-24 of m k between CTAs, and took a CTA of masked
// logits around -1e10 to an infinite sum.)  Temperatures outside [2^-40, 2^40] and maxima whose
// quotient is near fp32's upper end divide each difference instead; quotients that leave the range count as infinities.
//
// On B200, 128256 tokens: 576 rows with every rule 208 us (453 MB, 2.2 TB/s; a copy
// would take 69), 80 fp32 rows with masks and biases 45 us, one row 12 us, most of it the
// host's call (11 in a graph); 128 rows of 151936 tokens, on one CTA per SM with a few spilled words, 216 us (116 MB).  The long calls are bound by the rules' instructions and by a row's
// exchanges between its CTAs, with two CTAs per SM to hide them.  Earlier forms of the
// long one: entries in shared memory and a division for each 418 us; a cluster per row
// 324; clusters that stay, neighbouring tokens in one CTA 442, and dealt out in blocks 273.
#include "wal_kv8.cuh"

#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
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
  int B, T, V, share;  // entries per CTA, a multiple of 128
  int shift;           // log2 of the cluster's CTAs
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

constexpr float kLog2e = 1.4426950408889634f;

// Whether exp((x - top) / temp), x <= top, top not -inf, is ex2((x - top) * (kLog2e / temp)): differences that leave fp32's
// range count as 0 there, and no quotient is beyond its upper end.
__device__ __forceinline__ bool usual(float top, float temp) {
  return temp >= 9.0949470177292824e-13f && temp <= 1.099511627776e12f && top * (kLog2e / temp) < 1e30f;
}

// exp((x - top) / temp), x <= top, anywhere: quotients that leave fp32's range are infinities, and infinite ones equal.
__device__ __noinline__ float weight(float x, float top, float temp) {
  const float q = number(x / temp);
  if (q == -INFINITY) return 0.f;
  if (x == top) return 1.f;
  if (top / temp == INFINITY) return q == INFINITY ? 1.f : 0.f;
  const float half = top > 1e30f ? 0.5f : 1.f;  // the difference may pass the largest number
  return ex2((x * half - top * half) / temp * (kLog2e / half));
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
  // two in turn: what one CTA tells the others is read before any of them can be two exchanges further
  __shared__ float cmax[2][kMaxCluster], csum[2][kMaxCluster];
  __shared__ int cidx[2][kMaxCluster];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), ncta = (int)cl.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // entry i of this CTA is entry at(i) of the row; place(v) is where entry v is here, if it is
  auto at = [&](int i) { return ((i >> 7 << p.shift) + rank) << 7 | (i & 127); };
  auto place = [&](unsigned v) -> unsigned {
    return v < (unsigned)p.V && ((v >> 7) & (unsigned)(ncta - 1)) == (unsigned)rank ? (v >> 7 >> p.shift) << 7 | (v & 127) : 0xffffffffu;
  };
  const int v0 = at(4 * tid), step = NT / 32 << p.shift << 7;  // this thread's group k starts at entry v0 + k * step
  const bool counted = p.r.repetition || p.r.presence || p.r.frequency;
  const int nb = (int)p.r.num_bias;
  const int clusters = (int)gridDim.x / ncta, mine = (int)blockIdx.x / ncta, rows = p.B * p.T;
  const int row0 = (int)((long long)rows * mine / clusters), row1 = (int)((long long)rows * (mine + 1) / clusters);
  wal_kv8::chain();
  cl.sync();  // a CTA's shared memory may be written by the others once it has started
  int turn = 1;  // changes with each row that exchanges: skipped ones have no barrier
  int held = -1, upto = 0;  // the sequence whose words are there, and how much of its text they count
  for (int row = row0; row < row1; ++row) {
    const int b = row / p.T, t = row - b * p.T;
    float* const out = p.out + b * p.out_seq + t * p.out_row;
    auto write = [&](int k, const float (&x)[4]) {
      const int v = v0 + k * step;
      if (VEC) {
        if (v < p.V) __stcs(reinterpret_cast<float4*>(out + v), make_float4(x[0], x[1], x[2], x[3]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (v + e < p.V) out[v + e] = x[e];
      }
    };
    if (p.r.new_lens && t >= p.r.new_lens[b]) {  // for all CTAs of the row
      const float none[4] = {0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < K; ++k) write(k, none);
      continue;
    }
    float x[K][4];
    const long long base = b * p.ld_seq + t * p.ld_row;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int v = v0 + k * step;
      if (VEC) {
        const float4 f = v < p.V ? load4<DT>(p.logits, base + v) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        x[k][0] = f.x, x[k][1] = f.y, x[k][2] = f.z, x[k][3] = f.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k][e] = v + e < p.V ? load1<DT>(p.logits, base + v + e) : -INFINITY;
      }
    }
    if (row + 1 < row1) {
      const int nb2 = (row + 1) / p.T, nt = row + 1 - nb2 * p.T;
      constexpr int kLine = 128 / (DT == WAL_F32 ? 4 : 2);
      const long long first = nb2 * p.ld_seq + nt * p.ld_row;
      for (int i = kLine * tid; i < p.share && at(i) < p.V; i += kLine * NT) {
        const char* line = static_cast<const char*>(p.logits) + (first + at(i)) * (DT == WAL_F32 ? 4 : 2);
        asm volatile("prefetch.global.L2 [%0];" ::"l"(line));
      }
    }
    if ((counted || nb) && held != b) {
      __syncthreads();  // the words of the sequence before have been read
      for (int i = tid; i < p.share / 4; i += NT) reinterpret_cast<uint4*>(words)[i] = make_uint4(0u, 0u, 0u, 0u);
      for (int i = tid; i < nb; i += NT) {
        ids[i] = p.r.bias_ids[(long long)b * nb + i];
        adds[i] = p.r.bias[(long long)b * nb + i];
      }
      __syncthreads();
      if (counted) {
        const int* text = p.r.text + b * p.r.ld_text;
        upto = (int)min((long long)max(p.r.lens[b], -1 - t) + t + 1, (long long)p.r.text_len);
        const int prompt = p.r.prompt_lens ? p.r.prompt_lens[b] : 0;
#pragma unroll 4
        for (int j = tid; j < upto; j += NT) {
          const unsigned w = place((unsigned)text[j]);
          if (w != 0xffffffffu) {
            if (j < prompt) atomicOr(words + w, kPrompt);
            else atomicAdd(words + w, 1u);
          }
        }
      }
      float sum = 0.f;
      for (int i = tid; i < nb; i += NT) {
        const unsigned w = place((unsigned)ids[i]);
        if (w == 0xffffffffu) continue;
        bool first = true;
        for (int j = 0; j < i && first; ++j) first = ids[j] != ids[i];
        if (!first) continue;  // the first of equal ones adds them all, in order
        sum = adds[i];
        for (int j = i + 1; j < nb; ++j)
          if (ids[j] == ids[i]) sum += adds[j];
        atomicOr(words + w, (unsigned)(i + 1) << kBiasBit);
        if (sum != adds[i]) adds[i] = sum;  // no other thread reads the first one's
      }
      held = b;
      __syncthreads();
    } else if (counted) {  // the row's own token, if the text has it
      const int now = (int)min((long long)max(p.r.lens[b], -1 - t) + t + 1, (long long)p.r.text_len);
      __syncthreads();
      if (tid == 0 && now > upto) {
        const unsigned w = place((unsigned)p.r.text[b * p.r.ld_text + now - 1]);
        const int prompt = p.r.prompt_lens ? p.r.prompt_lens[b] : 0;
        if (w != 0xffffffffu) words[w] = now - 1 < prompt ? words[w] | kPrompt : words[w] + 1u;
      }
      upto = now;
      __syncthreads();
    }
    const float rep = p.r.repetition ? p.r.repetition[b] : 1.f, pres = p.r.presence ? p.r.presence[b] : 0.f;
    const float freq = p.r.frequency ? p.r.frequency[b] : 0.f, temp = p.r.temperature ? p.r.temperature[b] : 1.f;
    const bool greedy = !(temp > 0.f);
    const int* const mask = p.r.mask ? p.r.mask + b * p.r.mask_seq + t * p.r.mask_row : nullptr;
    // The nearest fp32 number to x / rep, so that what is equal by the definition stays equal: the product in 64 bits is off by
    // 2^-52, and a quotient of two 24-bit numbers is no border between fp32 numbers nor within 2^-49 of one (below
    // the normal numbers, where it can be, the last bit may differ).  576 rows of 128256 tokens: 207 us, 220 with a division.
    const double inv = 1.0 / (double)rep;
    if (counted || nb) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int i = 4 * (tid + NT * k);
        if (i >= p.share) break;
        const uint4 c = *reinterpret_cast<const uint4*>(words + i);
        const unsigned w[4] = {c.x, c.y, c.z, c.w}, any = c.x | c.y | c.z | c.w;
        if (any == 0u) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = x[k][e] > 0.f ? (float)((double)x[k][e] * inv) : x[k][e] * rep;
          const float z = y - freq * (float)(w[e] & kCount) - pres;
          x[k][e] = w[e] & kCount ? z : w[e] & kPrompt ? y : x[k][e];
        }
        if (any >> kBiasBit)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (w[e] >> kBiasBit) x[k][e] += adds[(w[e] >> kBiasBit) - 1];
      }
    }
    if (mask) {
      const int* const mine = mask + (v0 >> 5);  // groups of a thread have the same place in their words
      unsigned bits[K];
#pragma unroll
      for (int k = 0; k < K; ++k) bits[k] = v0 + k * step < p.V ? (unsigned)__ldg(mine + k * (step >> 5)) >> (v0 & 31) : 0u;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k][e] = (bits[k] >> e) & 1 ? x[k][e] : -INFINITY;
    }
    if (p.softmax && temp > FLT_MAX) {  // an infinite logit over an infinite temperature is no number
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k][e] = fabsf(x[k][e]) <= FLT_MAX ? x[k][e] : -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[k][e] = number(x[k][e]);
        top = fmaxf(top, x[k][e]);
      }
    if (!p.softmax) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!greedy && p.r.temperature)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[k][e] = number(x[k][e] / temp);
        write(k, x[k]);
      }
      continue;
    }
    turn ^= 1;
    // this CTA's largest, and its sum relative to it
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) wv[warp] = top;
    __syncthreads();
    top = wv[lane % W];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float scale = kLog2e / temp;
    float sum = 0.f;
    int where = 0x7fffffff;
    if (greedy) {
#pragma unroll
      for (int k = K - 1; k >= 0; --k)
#pragma unroll
        for (int e = 3; e >= 0; --e)
          if (x[k][e] == top) where = v0 + k * step + e;
    } else if (top > -INFINITY && usual(top, temp)) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[k][e] = ex2((x[k][e] - top) * scale);
          sum += x[k][e];
        }
    } else if (top > -INFINITY) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[k][e] = weight(x[k][e], top, temp);
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
    if (warp == 0) {
      float total = lane < W ? wsum[lane] : 0.f;
      int first = wi[lane % W];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
      }
      if (lane < ncta) {
        *cl.map_shared_rank(&cmax[turn][rank], lane) = top;
        *cl.map_shared_rank(&csum[turn][rank], lane) = total;
        *cl.map_shared_rank(&cidx[turn][rank], lane) = first;
      }
    }
    cl.sync();
    // a lane per CTA (the lanes beyond repeat them): the cluster's largest, and its sum relative to it
    const float its = cmax[turn][lane & (ncta - 1)];
    float all = its;
    int best = cidx[turn][lane & (ncta - 1)];
#pragma unroll
    for (int o = kMaxCluster / 2; o > 0; o >>= 1)
      better(all, best, __shfl_xor_sync(0xffffffffu, all, o), __shfl_xor_sync(0xffffffffu, best, o));
    const bool near = usual(all, temp) && usual(-all, temp);  // nor beyond the lower one, where nothing is left of the row
    auto relative = [&](float m) { return near ? ex2((m - all) * scale) : weight(m, all, temp); };
    float total = lane < ncta ? csum[turn][lane & (ncta - 1)] * relative(its) : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    // a CTA with nothing left has entries of -inf, which are not multiplied
    const float factor = greedy || !(total > 0.f) || top == -INFINITY ? 0.f : relative(top) / total;
    const int one = greedy && all > -INFINITY ? best : -1;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (factor == 0.f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k][e] = v0 + k * step + e == one ? 1.f : 0.f;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k][e] *= factor;
      }
      write(k, x[k]);
    }
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
  // what eight GPCs of 16 to 18 SMs hold of clusters of eight
  const int resident = std::max(1, 128 * (NT == 512 ? 2 : 1) / cluster);
  return wal_kv8::launch_chain(kern, dim3((unsigned)(std::min(p.B * p.T, resident) * cluster)), NT, words ? p.share * 4 : 0, st, p, cluster);
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
  p.share = (int)((V + 128 * cluster - 1) / (128 * cluster)) * 128;
  p.shift = cluster == 8 ? 3 : cluster == 4 ? 2 : cluster == 2 ? 1 : 0;
  const bool vec = V % 4 == 0 && ld_row % 4 == 0 && ld_seq % 4 == 0 && out_row % 4 == 0 && out_seq % 4 == 0 &&
                   !((uintptr_t)logits & (4 * size - 1)) && !((uintptr_t)out & 15);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == WAL_BF16) return launch_type<WAL_BF16>(p, vec, cluster, st);
  if (dtype == WAL_F16) return launch_type<WAL_F16>(p, vec, cluster, st);
  return launch_type<WAL_F32>(p, vec, cluster, st);
}

}  // extern "C"
