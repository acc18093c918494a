// Shared parts of the paged 8-bit KV cache kernels: the cache view, the page
// lookup and the two 8-bit code types.
//
// A value is code * scale with one fp32 scale per (page, kv head) of K and of
// V.  int8 codes are the integers -127..127, e4m3 codes the finite 8-bit
// floats up to 448; both are reached by clamping x / scale and rounding to
// nearest even, so a code never stands for an infinity or a NaN.
#pragma once
#include "../../include/wal_rvq.h"

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace wal_kv8 {

// One layer's half (K or V) of the cache: codes [pages][hkv][P][hd], scales [pages][hkv].
struct LayerView {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
};

__host__ __device__ inline long long half_codes(const wal_kv8_cache& c) {
  return (long long)c.num_pages * c.kv_heads * c.page_size * c.head_dim;
}
__host__ __device__ inline long long half_scales(const wal_kv8_cache& c) { return (long long)c.num_pages * c.kv_heads; }

inline LayerView layer_view(const wal_kv8_cache& c, int layer) {
  LayerView v;
  v.k = static_cast<uint8_t*>(c.codes) + 2 * layer * half_codes(c);
  v.v = v.k + half_codes(c);
  v.ks = c.scales + 2 * layer * half_scales(c);
  v.vs = v.ks + half_scales(c);
  return v;
}

// Argument check shared by the entry points.
inline int check_cache(const wal_kv8_cache* c, int layer) {
  if (!c || !c->codes || !c->scales) return WAL_ERR_INVALID_ARGUMENT;
  if (c->num_pages <= 0 || c->num_pages > 0x7fffffff || c->layers <= 0 || c->kv_heads <= 0 || c->kv_heads > 65535)
    return WAL_ERR_SHAPE;
  if (layer < 0 || layer >= c->layers) return WAL_ERR_SHAPE;
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64) return WAL_ERR_UNSUPPORTED;
  if (c->head_dim != 64 && c->head_dim != 128) return WAL_ERR_UNSUPPORTED;
  if (c->kind != WAL_KV_INT8 && c->kind != WAL_KV_E4M3) return WAL_ERR_UNSUPPORTED;
  if (((uintptr_t)c->codes & 15) || ((uintptr_t)c->scales & 3)) return WAL_ERR_ALIGNMENT;
  return WAL_OK;
}

template <int KIND>
__device__ __forceinline__ float qmax() {
  return KIND == WAL_KV_INT8 ? 127.f : 448.f;
}

// The four codes of a word as fp32.
template <int KIND>
__device__ __forceinline__ void decode4(uint32_t w, float (&f)[4]) {
  if (KIND == WAL_KV_INT8) {
    // byte u = code + 128 in the fraction of 2^23: a logic instruction and an exact subtraction (a conversion runs at a quarter of the rate)
    const uint32_t u = w ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7650 + i)) - 8388736.f;
  } else {
    const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
    f[0] = a.x;
    f[1] = a.y;
    f[2] = b.x;
    f[3] = b.y;
  }
}

// round(clamp(x)) as a code; x is already divided by the scale.  NaN -> 0.
template <int KIND>
__device__ __forceinline__ uint32_t encode(float x) {
  if (!(x == x)) return 0u;
  x = fminf(fmaxf(x, -qmax<KIND>()), qmax<KIND>());
  if (KIND == WAL_KV_INT8) return (uint32_t)__float2int_rn(x) & 0xffu;
  return (uint32_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

// Page of a table entry, -1 where the entry names none.
__device__ __forceinline__ int valid_page(int e, int pages) { return (unsigned)e < (unsigned)pages ? e : -1; }

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t v;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  return v;
}

// Programmatic dependent launch: a kernel waits for the grids before it in the
// stream before it touches memory, and lets the next one start launching.
__device__ __forceinline__ void chain() {
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
}

constexpr int kMaxDevices = 64;

// SM count of the current device, looked up once per device.
inline int sm_count() {
  static std::atomic<int> known[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 148;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Launches kern(p) in the chain.
template <typename Kern, typename Params>
int launch_chain(Kern kern, dim3 grid, int threads, int smem, cudaStream_t stream, const Params& p, int cluster = 0) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)(cluster > 0 ? cluster : 1);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kern, p) != cudaSuccess) return WAL_ERR_CUDA;
  return cudaGetLastError() == cudaSuccess ? WAL_OK : WAL_ERR_CUDA;
}

}  // namespace wal_kv8
