// Attention of new tokens over the paged 8-bit KV cache (grouped-query heads).
//
//   out[b, t, h] = sum_j softmax_j(scale * q[b, t, h] . k_j) v_j,  j <= lens[b] + t
//
// One CTA per query row; its warps take positions in turn, each with a running
// maximum and sum (softmax in one pass), joined at the end.
#include "wal_kv8.cuh"

namespace {

using namespace wal_kv8;

constexpr int kThreads = 256;

struct AttnParams {
  const uint16_t* q;
  long long ld_q;
  LayerView kv;
  int T, hq, hkv, P, pages, max_pages;
  const int* table;
  long long ld_table;
  const int* lens;
  const int* new_lens;
  float qscale;  // scale * log2(e)
  uint16_t* out;
  long long ld_out;
};

template <int HD, int KIND>
__global__ void __launch_bounds__(kThreads) kv8_attention_kernel(const __grid_constant__ AttnParams p) {
  constexpr int NW = kThreads / 32, E = HD / 32;
  __shared__ float sm[NW], sl[NW], so[NW][HD];
  const int h = blockIdx.x % p.hq, m = blockIdx.x / p.hq, b = m / p.T, t = m - b * p.T;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kvh = h / (p.hq / p.hkv);
  const int nn = p.new_lens ? min(p.new_lens[b], p.T) : p.T;
  uint16_t* orow = p.out + (long long)m * p.ld_out + (long long)h * HD;
  const long long cap = (long long)p.max_pages * p.P;
  const int n = t < nn ? (int)min((long long)max(p.lens[b], 0) + t + 1, cap) : 0;
  float q[E], o[E], mx = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __uint_as_float((uint32_t)p.q[(long long)m * p.ld_q + (long long)h * HD + e * 32 + lane] << 16);
    o[e] = 0.f;
  }
  for (int j = warp; j < n; j += NW) {
    const int page = valid_page(p.table[(long long)b * p.ld_table + j / p.P], p.pages);
    if (page < 0) continue;
    const long long blk = (long long)page * p.hkv + kvh, row = (blk * p.P + j % p.P) * HD;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], decode<KIND>(p.kv.k[row + e * 32 + lane]), s);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
    s *= p.kv.ks[blk] * p.qscale;
    const float mn = fmaxf(mx, s), al = mx == -INFINITY ? 0.f : exp2f(mx - mn), w = exp2f(s - mn);
    const float wv = w * p.kv.vs[blk];
    l = fmaf(l, al, w);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], al, wv * decode<KIND>(p.kv.v[row + e * 32 + lane]));
    mx = mn;
  }
  if (lane == 0) sm[warp] = mx, sl[warp] = l;
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][e * 32 + lane] = o[e];
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < NW; ++w) M = fmaxf(M, sm[w]);
  for (int w = 0; w < NW; ++w)
    if (sm[w] != -INFINITY) L = fmaf(exp2f(sm[w] - M), sl[w], L);
  for (int d = threadIdx.x; d < HD; d += kThreads) {
    float a = 0.f;
    for (int w = 0; w < NW; ++w)
      if (sm[w] != -INFINITY) a = fmaf(exp2f(sm[w] - M), so[w][d], a);
    orow[d] = __bfloat16_as_ushort(__float2bfloat16_rn(L > 0.f ? a / L : 0.f));
  }
}

}  // namespace

extern "C" {

size_t wal_kv8_attention_workspace(const wal_kv8_cache* cache, int64_t B, int64_t T, int32_t hq) {
  if (!cache || cache->kv_heads <= 0 || B <= 0 || T <= 0 || hq <= 0 || hq % cache->kv_heads) return 0;
  return 256;
}

int wal_kv8_attention(const wal_kv8_cache* cache, int32_t layer, const uint16_t* q, int64_t ld_q, int64_t B, int64_t T,
                      int32_t hq, const int32_t* table, int64_t ld_table, int64_t max_pages, const int32_t* lens,
                      const int32_t* new_lens, float scale, uint16_t* out, int64_t ld_out, void* workspace,
                      size_t workspace_bytes, void* stream) {
  int st = check_cache(cache, layer);
  if (st != WAL_OK) return st;
  if (!q || !table || !lens || !out || !workspace) return WAL_ERR_INVALID_ARGUMENT;
  if (B <= 0 || T <= 0 || hq <= 0 || hq % cache->kv_heads || max_pages <= 0 || ld_table < max_pages) return WAL_ERR_SHAPE;
  const int hd = cache->head_dim;
  if (B > 0x7fffffff || T > 0x7fffffff || max_pages > 0x7fffffff / cache->page_size || B * T > 0x7fffffff / hq) return WAL_ERR_SHAPE;
  if (ld_q < (int64_t)hq * hd || ld_out < (int64_t)hq * hd) return WAL_ERR_SHAPE;
  if (((uintptr_t)q & 15) || ((uintptr_t)out & 15) || ((uintptr_t)workspace & 255) || (ld_q % 8) || (ld_out % 8)) return WAL_ERR_ALIGNMENT;
  if (workspace_bytes < wal_kv8_attention_workspace(cache, B, T, hq)) return WAL_ERR_BUFFER_TOO_SMALL;
  AttnParams p = {q, ld_q, layer_view(*cache, layer), (int)T, hq, cache->kv_heads, cache->page_size, (int)cache->num_pages,
                  (int)max_pages, table, ld_table, lens, new_lens, scale * 1.4426950408889634f, out, ld_out};
  const unsigned grid = (unsigned)(B * T * hq);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (hd == 128) {
    if (cache->kind == WAL_KV_INT8) kv8_attention_kernel<128, WAL_KV_INT8><<<grid, kThreads, 0, s>>>(p);
    else kv8_attention_kernel<128, WAL_KV_E4M3><<<grid, kThreads, 0, s>>>(p);
  } else {
    if (cache->kind == WAL_KV_INT8) kv8_attention_kernel<64, WAL_KV_INT8><<<grid, kThreads, 0, s>>>(p);
    else kv8_attention_kernel<64, WAL_KV_E4M3><<<grid, kThreads, 0, s>>>(p);
  }
  return launch_status();
}

}  // extern "C"
