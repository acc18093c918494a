// Store and read-back of the paged 8-bit KV cache.
//
//   kv8_append_kernel  rotary positions of q and k, and the new tokens of every
//                      sequence into their pages.  A CTA owns one (sequence,
//                      touched page, kv head) of K or of V: it reads its new
//                      values, takes their largest magnitude a, sets the block's
//                      scale to max(old, a * (1 / Q)), re-rounds the earlier codes
//                      of the block where the scale grew, and stores the codes.
//                      No other CTA touches the block, so the result has one
//                      order; a page's values stay in registers between the
//                      maximum and the codes.  Further CTAs rotate q, a warp per
//                      token and group of heads that share one load of angles.
//                      Rotation rounds each product and sum in fp32; K is rounded
//                      once, from fp32 to its code.
//   kv8_read_kernel    values code * scale of a range of positions.
//
// Bounds, on B200: four prompts of 1270 tokens on average (64 query and 8 kv heads of 128; 8192 rows
// with padding): append 54 us for 277 MB, 5.1 TB/s or 78% of a copy's rate, of which
// 265 MB are q and qkv; read-back 13 us for 48 MB.  A decode step of three
// sequences takes 4.3 us for both kernels, all of it launch and two dependent
// loads.  Threads per CTA and CTAs per SM: 256 and 3 against 128 and 5 made no
// difference to the whole (68 us); fewer looping query warps lose (72 us with 3
// CTAs per SM, 68 with 16).
#include "wal_kv8.cuh"

namespace {

using namespace wal_kv8;

struct AppendParams {
  const uint16_t* qkv;
  long long ld;
  int B, T, hq, hkv, pages, max_pages, touched;
  const int* table;
  long long ld_table;
  const int* lens;
  const int* new_lens;
  const float* cos;
  const float* sin;
  int max_pos;
  uint16_t* q_out;
  long long ld_q;
  LayerView kv;
  unsigned kv_ctas;  // CTAs of the K/V part, before those of q
  unsigned q_items;  // (token, group of heads) pairs
};

// 16 values of one token and head: dims [8c, 8c + 8) and their rotation partners hd/2 later.
struct Pair {
  float a[8], b[8];
};

__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
  f[0] = bf16_lo(v.x); f[1] = bf16_hi(v.x); f[2] = bf16_lo(v.y); f[3] = bf16_hi(v.y);
  f[4] = bf16_lo(v.z); f[5] = bf16_hi(v.z); f[6] = bf16_lo(v.w); f[7] = bf16_hi(v.w);
}

struct Raw {
  uint4 a, b;
};

template <int HD>
__device__ __forceinline__ Raw load_raw(const uint16_t* src, int c) {
  return {__ldg(reinterpret_cast<const uint4*>(src + 8 * c)), __ldg(reinterpret_cast<const uint4*>(src + HD / 2 + 8 * c))};
}

__device__ __forceinline__ Pair widen(const Raw& r) {
  Pair p;
  unpack(r.a, p.a);
  unpack(r.b, p.b);
  return p;
}

// Cosines and sines of the angles of dims [8c, 8c + 8) at a position.
struct Angles {
  float c[8], s[8];
};

template <int HD>
__device__ __forceinline__ Angles load_angles(const float* cos, const float* sin, int pos, int c) {
  Angles g;
  const float4* cp = reinterpret_cast<const float4*>(cos + (long long)pos * (HD / 2) + 8 * c);
  const float4* sp = reinterpret_cast<const float4*>(sin + (long long)pos * (HD / 2) + 8 * c);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    *reinterpret_cast<float4*>(g.c + 4 * h) = __ldg(cp + h);
    *reinterpret_cast<float4*>(g.s + 4 * h) = __ldg(sp + h);
  }
  return g;
}

__device__ __forceinline__ void rotate(Pair& p, const Angles& g) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = p.a[i], y = p.b[i];
    p.a[i] = __fadd_rn(__fmul_rn(x, g.c[i]), __fmul_rn(-y, g.s[i]));
    p.b[i] = __fadd_rn(__fmul_rn(y, g.c[i]), __fmul_rn(x, g.s[i]));
  }
}

template <int KIND>
__device__ __forceinline__ uint2 encode8(const float (&x)[8], float s) {
  uint32_t w[2] = {0u, 0u};
  if (s > 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i >> 2] |= encode<KIND>(__fdiv_rn(x[i], s)) << (8 * (i & 3));
  }
  return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}

constexpr int kThreads = 256;       // append
constexpr int kReadThreads = 128;

// Query heads that a warp rotates.
template <int HD>
__host__ __device__ constexpr int kHeads() {
  return 4 * 32 / (HD / 16);
}

template <int HD, int P, int KIND>
__global__ void __launch_bounds__(kThreads, 3) kv8_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr int C = HD / 16;                              // 16-value pieces per token and head
  constexpr int IT = (P * C + kThreads - 1) / kThreads;   // pieces per thread of a whole page
  const int tid = threadIdx.x;
  chain();
  if (blockIdx.x >= p.kv_ctas) {  // q rows: a warp rotates up to kHeads heads of one token by one load of its angles
    constexpr int H = 32 / C, kIter = kHeads<HD>() / H;
    const int lane = tid & 31, c = lane % C;
    const unsigned groups = (unsigned)(p.hq + kHeads<HD>() - 1) / kHeads<HD>(), warps = (gridDim.x - p.kv_ctas) * (kThreads / 32);
    for (unsigned w = (blockIdx.x - p.kv_ctas) * (kThreads / 32) + (tid >> 5); w < p.q_items; w += warps) {
      const unsigned m = w / groups, h0 = (w - m * groups) * kHeads<HD>() + lane / C;
      const int b = (int)m / p.T, t = (int)m - b * p.T;
      const int nn = p.new_lens ? min(p.new_lens[b], p.T) : p.T;
      const long long pos = (long long)max(p.lens[b], 0) + t;
      const bool real = t < nn && (!p.cos || pos < p.max_pos);
      const uint16_t* src = p.qkv + (long long)m * p.ld + h0 * HD;
      uint16_t* dst = p.q_out + (long long)m * p.ld_q + h0 * HD + 8 * c;
      Raw raw[kIter];
#pragma unroll
      for (int i = 0; i < kIter; ++i)
        if (real && h0 + i * H < (unsigned)p.hq) raw[i] = load_raw<HD>(src + i * H * HD, c);
      Angles g;
      if (real && p.cos) g = load_angles<HD>(p.cos, p.sin, (int)pos, c);
#pragma unroll
      for (int i = 0; i < kIter; ++i) {
        if (h0 + i * H >= (unsigned)p.hq) break;
        uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
        if (real) {
          Pair x = widen(raw[i]);
          if (p.cos) rotate(x, g);
          lo = make_uint4(pack_bf16(x.a[0], x.a[1]), pack_bf16(x.a[2], x.a[3]), pack_bf16(x.a[4], x.a[5]), pack_bf16(x.a[6], x.a[7]));
          hi = make_uint4(pack_bf16(x.b[0], x.b[1]), pack_bf16(x.b[2], x.b[3]), pack_bf16(x.b[4], x.b[5]), pack_bf16(x.b[6], x.b[7]));
        }
        *reinterpret_cast<uint4*>(dst + i * H * HD) = lo;
        *reinterpret_cast<uint4*>(dst + i * H * HD + HD / 2) = hi;
      }
    }
    return;
  }
  const int kv = blockIdx.x & 1;
  unsigned u = blockIdx.x >> 1;
  const int h = (int)(u % p.hkv);
  u /= p.hkv;
  const int j = (int)(u % p.touched), b = (int)(u / p.touched);
  const int len = max(p.lens[b], 0);
  int nn = p.new_lens ? min(p.new_lens[b], p.T) : p.T;
  const long long pg = (long long)(len / P) + j;  // page of the sequence
  if (pg >= p.max_pages) return;
  const long long start = pg * P;
  // new tokens t in [t0, t1) fall into this page, at slots start + ...
  long long t0 = start > len ? start - len : 0, t1 = start + P - len;
  if (t1 > nn) t1 = nn;
  if (p.cos && t1 > (long long)p.max_pos - len) t1 = (long long)p.max_pos - len;
  if (t0 >= t1) return;
  const int page = valid_page(p.table[(long long)b * p.ld_table + pg], p.pages);
  if (page < 0) return;
  const int slot0 = (int)(len + t0 - start), cnt = (int)(t1 - t0);  // slots [slot0, slot0 + cnt)
  const uint16_t* src = p.qkv + ((long long)b * p.T + t0) * p.ld + (long long)(p.hq + kv * p.hkv + h) * HD;
  Raw raw[IT];
  Pair x[IT];
  float a = 0.f;
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int i = it * kThreads + tid, t = i / C, c = i % C;
    if (t < cnt) raw[it] = load_raw<HD>(src + (long long)t * p.ld, c);
  }
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int i = it * kThreads + tid, t = i / C, c = i % C;
    if (t < cnt) {
      x[it] = widen(raw[it]);
      if (kv == 0 && p.cos) rotate(x[it], load_angles<HD>(p.cos, p.sin, (int)(len + t0) + t, c));
#pragma unroll
      for (int e = 0; e < 8; ++e) a = fmaxf(a, fmaxf(finite_abs(x[it].a[e]), finite_abs(x[it].b[e])));
    }
  }
  __shared__ float red[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  if ((tid & 31) == 0) red[tid >> 5] = a;
  float* scale = (kv == 0 ? p.kv.ks : p.kv.vs) + (long long)page * p.hkv + h;
  const float s0 = slot0 > 0 ? *scale : 0.f;
  __syncthreads();  // every thread has read the old scale
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) a = fmaxf(a, red[w]);
  const float s = fmaxf(s0, __fmul_rn(a, 1.f / qmax<KIND>()));
  uint8_t* blk = (kv == 0 ? p.kv.k : p.kv.v) + ((long long)page * p.hkv + h) * (P * HD);
  if (s > s0 && slot0 > 0) {  // the scale grew: earlier codes in units of the new one
    const float r = __fdiv_rn(s0, s);
    for (int i = tid; i < slot0 * (HD / 4); i += kThreads) {
      uint32_t* w = reinterpret_cast<uint32_t*>(blk) + i;
      const uint32_t v = *w;
      float f[4];
      decode4<KIND>(v, f);
      uint32_t n = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) n |= encode<KIND>(__fmul_rn(f[e], r)) << (8 * e);
      *w = n;
    }
  }
  if (tid == 0) *scale = s;
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int i = it * kThreads + tid, t = i / C, c = i % C;
    if (t < cnt) {
      uint8_t* row = blk + (slot0 + t) * HD + 8 * c;
      *reinterpret_cast<uint2*>(row) = encode8<KIND>(x[it].a, s);
      *reinterpret_cast<uint2*>(row + HD / 2) = encode8<KIND>(x[it].b, s);
    }
  }
}

struct ReadParams {
  LayerView kv;
  int B, hkv, pages, max_pages;
  long long L;
  unsigned chunks;  // CTAs per (sequence, kv head) of K or V
  const int* table;
  long long ld_table;
  const int* first;
  const int* count;
  void* k_out;
  void* v_out;
};

// A CTA reads kReadRows positions of one (sequence, kv head) of K or V, 16 codes per thread at a time.
constexpr int kReadRows = 64;

template <int HD, int P, int KIND, bool F32>
__global__ void __launch_bounds__(kReadThreads) kv8_read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int C = HD / 16, STEP = kReadThreads / C;
  chain();
  const unsigned u = blockIdx.x / p.chunks, chunk = blockIdx.x - u * p.chunks, kv = u & 1, bh = u >> 1;
  const int b = (int)(bh / p.hkv), h = (int)(bh - b * p.hkv), c = threadIdx.x % C;
  const int count = p.count[b];
  const long long first = max(p.first[b], 0);
  const uint8_t* codes = (kv ? p.kv.v : p.kv.k) + (long long)h * (P * HD) + 16 * c;
  const float* scales = (kv ? p.kv.vs : p.kv.ks) + h;
  uint4 w[kReadRows / STEP];
  float s[kReadRows / STEP];
#pragma unroll
  for (int i = 0; i < kReadRows / STEP; ++i) {
    const int l = (int)chunk * kReadRows + i * STEP + threadIdx.x / C;
    const long long pos = first + l;
    w[i] = make_uint4(0u, 0u, 0u, 0u);
    s[i] = 0.f;
    if (l < count && l < p.L && pos / P < p.max_pages) {
      const int page = valid_page(p.table[(long long)b * p.ld_table + pos / P], p.pages);
      if (page >= 0) {
        s[i] = scales[(long long)page * p.hkv];
        w[i] = *reinterpret_cast<const uint4*>(codes + (long long)page * p.hkv * (P * HD) + (int)(pos % P) * HD);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kReadRows / STEP; ++i) {
    const int l = (int)chunk * kReadRows + i * STEP + threadIdx.x / C;
    if (l >= p.L) break;
    const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
    float f[16];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float g[4];
      decode4<KIND>(x[e], g);
#pragma unroll
      for (int y = 0; y < 4; ++y) f[4 * e + y] = __fmul_rn(g[y], s[i]);
    }
    const long long at = ((long long)bh * p.L + l) * HD + 16 * c;
    if (F32) {
      float4* dst = reinterpret_cast<float4*>(static_cast<float*>(kv ? p.v_out : p.k_out) + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[e] = make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
    } else {
      uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(kv ? p.v_out : p.k_out) + at);
#pragma unroll
      for (int e = 0; e < 2; ++e)
        dst[e] = make_uint4(pack_bf16(f[8 * e], f[8 * e + 1]), pack_bf16(f[8 * e + 2], f[8 * e + 3]),
                            pack_bf16(f[8 * e + 4], f[8 * e + 5]), pack_bf16(f[8 * e + 6], f[8 * e + 7]));
    }
  }
}

template <int HD, int P, int KIND>
int launch_append(const AppendParams& p, unsigned grid, cudaStream_t st) {
  return launch_chain(kv8_append_kernel<HD, P, KIND>, dim3(grid), kThreads, 0, st, p);
}

template <int HD, int P, int KIND>
int launch_read(const ReadParams& p, bool f32, unsigned grid, cudaStream_t st) {
  if (f32) return launch_chain(kv8_read_kernel<HD, P, KIND, true>, dim3(grid), kReadThreads, 0, st, p);
  return launch_chain(kv8_read_kernel<HD, P, KIND, false>, dim3(grid), kReadThreads, 0, st, p);
}

// Calls F<HD, P, KIND>(args...) for the cache's shape (check_cache has passed).
#define WAL_KV8_DISPATCH(c, F, ...)                                                                   \
  do {                                                                                                \
    const int key_ = ((c)->head_dim == 128 ? 6 : 0) + ((c)->page_size == 16 ? 0 : (c)->page_size == 32 ? 2 : 4) + \
                     ((c)->kind == WAL_KV_E4M3 ? 1 : 0);                                              \
    switch (key_) {                                                                                   \
      case 0: return F<64, 16, WAL_KV_INT8>(__VA_ARGS__);                                             \
      case 1: return F<64, 16, WAL_KV_E4M3>(__VA_ARGS__);                                             \
      case 2: return F<64, 32, WAL_KV_INT8>(__VA_ARGS__);                                             \
      case 3: return F<64, 32, WAL_KV_E4M3>(__VA_ARGS__);                                             \
      case 4: return F<64, 64, WAL_KV_INT8>(__VA_ARGS__);                                             \
      case 5: return F<64, 64, WAL_KV_E4M3>(__VA_ARGS__);                                             \
      case 6: return F<128, 16, WAL_KV_INT8>(__VA_ARGS__);                                            \
      case 7: return F<128, 16, WAL_KV_E4M3>(__VA_ARGS__);                                            \
      case 8: return F<128, 32, WAL_KV_INT8>(__VA_ARGS__);                                            \
      case 9: return F<128, 32, WAL_KV_E4M3>(__VA_ARGS__);                                            \
      case 10: return F<128, 64, WAL_KV_INT8>(__VA_ARGS__);                                           \
      default: return F<128, 64, WAL_KV_E4M3>(__VA_ARGS__);                                           \
    }                                                                                                 \
  } while (0)

}  // namespace

extern "C" {

int wal_kv8_append(const wal_kv8_cache* cache, int32_t layer, const uint16_t* qkv, int64_t ld_qkv, int64_t B, int64_t T,
                   int32_t hq, const int32_t* table, int64_t ld_table, int64_t max_pages, const int32_t* lens,
                   const int32_t* new_lens, const float* cos, const float* sin, int64_t max_pos, uint16_t* q_out,
                   int64_t ld_q, void* stream) {
  int st = check_cache(cache, layer);
  if (st != WAL_OK) return st;
  if (!qkv || !table || !lens || !q_out || !cos != !sin) return WAL_ERR_INVALID_ARGUMENT;
  if (B <= 0 || T <= 0 || hq <= 0 || hq % cache->kv_heads || max_pages <= 0 || ld_table < max_pages) return WAL_ERR_SHAPE;
  if (B > 0x7fffffff || T > 0x7fffffff || max_pages > 0x7fffffff / cache->page_size) return WAL_ERR_SHAPE;
  if (cos && (max_pos <= 0 || max_pos > 0x7fffffff)) return WAL_ERR_SHAPE;
  const int hd = cache->head_dim, P = cache->page_size;
  if (ld_qkv < (int64_t)(hq + 2 * cache->kv_heads) * hd || ld_q < (int64_t)hq * hd) return WAL_ERR_SHAPE;
  if (((uintptr_t)qkv & 15) || ((uintptr_t)q_out & 15) || ((uintptr_t)cos & 15) || ((uintptr_t)sin & 15) || (ld_qkv % 8) ||
      (ld_q % 8))
    return WAL_ERR_ALIGNMENT;
  AppendParams p = {};
  p.qkv = qkv;
  p.ld = ld_qkv;
  p.B = (int)B;
  p.T = (int)T;
  p.hq = hq;
  p.hkv = cache->kv_heads;
  p.pages = (int)cache->num_pages;
  p.max_pages = (int)max_pages;
  p.touched = (int)((T + P - 2) / P + 1);  // T tokens from any slot of a page
  p.table = table;
  p.ld_table = ld_table;
  p.lens = lens;
  p.new_lens = new_lens;
  p.cos = cos;
  p.sin = sin;
  p.max_pos = (int)max_pos;
  p.q_out = q_out;
  p.ld_q = ld_q;
  p.kv = layer_view(*cache, layer);
  const int heads = hd == 128 ? kHeads<128>() : kHeads<64>();
  if (B * T > 0x3fffffff / ((hq + heads - 1) / heads)) return WAL_ERR_SHAPE;
  const long long kv_ctas = 2LL * B * p.touched * p.hkv;
  p.q_items = (unsigned)(B * T * ((hq + heads - 1) / heads));
  const long long q_most = (p.q_items + kThreads / 32 - 1) / (kThreads / 32), q_ctas = q_most < 16LL * sm_count() ? q_most : 16LL * sm_count();
  if (kv_ctas + q_ctas > 0x7fffffff) return WAL_ERR_SHAPE;
  p.kv_ctas = (unsigned)kv_ctas;
  const unsigned grid = (unsigned)(kv_ctas + q_ctas);
  WAL_KV8_DISPATCH(cache, launch_append, p, grid, static_cast<cudaStream_t>(stream));
}

int wal_kv8_read(const wal_kv8_cache* cache, int32_t layer, int64_t B, const int32_t* table, int64_t ld_table,
                 int64_t max_pages, const int32_t* first, const int32_t* count, int64_t L, void* k_out, void* v_out,
                 int out_dtype, void* stream) {
  int st = check_cache(cache, layer);
  if (st != WAL_OK) return st;
  if (!table || !first || !count || !k_out || !v_out) return WAL_ERR_INVALID_ARGUMENT;
  if (out_dtype != WAL_F32 && out_dtype != WAL_BF16) return WAL_ERR_UNSUPPORTED;
  if (B <= 0 || L <= 0 || max_pages <= 0 || ld_table < max_pages) return WAL_ERR_SHAPE;
  if (B > 0x7fffffff || L > 0x7fffffff || max_pages > 0x7fffffff / cache->page_size) return WAL_ERR_SHAPE;
  if (((uintptr_t)k_out & 15) || ((uintptr_t)v_out & 15)) return WAL_ERR_ALIGNMENT;
  ReadParams p = {};
  p.kv = layer_view(*cache, layer);
  p.B = (int)B;
  p.hkv = cache->kv_heads;
  p.pages = (int)cache->num_pages;
  p.max_pages = (int)max_pages;
  p.L = L;
  p.table = table;
  p.ld_table = ld_table;
  p.first = first;
  p.count = count;
  p.k_out = k_out;
  p.v_out = v_out;
  p.chunks = (unsigned)((L + kReadRows - 1) / kReadRows);
  const long long units = 2LL * B * p.hkv;
  if (units > 0x7fffffff / p.chunks) return WAL_ERR_SHAPE;
  const unsigned grid = (unsigned)(units * p.chunks);
  WAL_KV8_DISPATCH(cache, launch_read, p, out_dtype == WAL_F32, grid, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
