// 4-bit linear with group scales: y = x W^T for up to 32 tokens per launch.
//
//   y[m, n] = sum_g s[n, g] * sum_{k in g} (c[n, k] - z[n, g]) * x[m, k] + bias[n]
//
// The codes are read once and are nearly all of the traffic, so the kernel is
// built to keep 16-byte loads of them in flight.  They are packed in the order of
// the A fragments of mma.sync m16n8k16 (16 weight rows; tokens are the eight
// columns): one 16-byte load of a warp is 16 rows x 64 columns, each of its words
// a lane's fragment of one product.  A code becomes a 16-bit float with a logic
// instruction (the code in the low bits of 128 as bf16, of 1024 as f16) and an exact
// subtraction of 128 + z or 1024 + z, so the products see whole numbers; a group's
// fp32 sum is scaled once.  The order of k inside a product is free: a lane's
// columns are chosen so that its activations are two 16-byte loads.
//
// Split.  CTAs that fill the GPU twice take groups of row tiles in turn, and keep
// the activations in shared memory for all of them, rows 64 bytes out of step so
// that the matrix fragments meet no bank twice; where they do not fit they are read
// through L1.  A warp takes a row tile and every ks-th chunk of 64
// columns, loading the next chunks, the next group's first ones among them, while
// it multiplies.  What the ks warps have of a tile is added in order, so results do
// not depend on timing.
//
// On B200: 128256 x 4096 for five tokens 75 us, 3.65 TB/s (its bytes at a copy's rate:
// 41).  In a graph, for sixteen tokens 119, for 32 217; 28672 x 4096 for one 23 (copy: 9);
// 4096 x 4096 for one 5.8; 4096 x 14336 for sixteen, with zero points, 18 (copy: 5).
// Bound by instructions: 23 for each fragment of 256 weights, of which unpacking takes
// eleven.  Not kept: two row tiles per warp for 9 to 16 tokens (126 against 118 at
// 128256 x 4096, 26 against 18 at 4096 x 14336, no different at 28672 x 4096); a
// cluster that splits the columns (37 against 18 at 4096 x 14336); activations as f16, whose
// longer fraction saves shifts (no gain, slower for one token).
#include "wal_kv8.cuh"

#include <cuda_fp16.h>

namespace {

using wal_kv8::kMaxDevices;
using wal_kv8::launch_chain;
using wal_kv8::sm_count;

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kAhead = 4;  // chunks loaded together

template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool F16>
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (F16) asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// 128 (bf16) or 1024 (f16) twice; a code in the low bits adds itself
template <bool F16>
__host__ __device__ __forceinline__ constexpr uint32_t magic() { return F16 ? 0x64006400u : 0x43004300u; }

// Passed as a parameter: a logic instruction takes one immediate, and two known constants cost a move each time.
struct Masks {
  uint32_t nibbles = 0x000f000fu, bf16 = magic<false>(), f16 = magic<true>();
};

struct Int4Params {
  const uint4* packed;    // [tiles][chunks][32]
  const uint32_t* scales; // [tiles][groups][8] pairs of rows r, r + 8
  const uint16_t* zeros;  // likewise, bytes
  const uint16_t* bias;
  const uint16_t* x;
  void* y;
  long long ldx, ldy;
  int M, N, K, tiles, chunks, groups;
  int per;  // chunks per group as a shift (0 or 1)
  int ks;   // warps that share a tile
  int stride;        // bytes between activation rows in shared memory
  int f16;           // activations
  Masks masks;
  int y_dtype;
};

// A fragment of one product from a word: rows r (registers 0, 2) and r + 8 (1, 3), minus their zero points.
template <bool F16>
__device__ __forceinline__ void unpack(const Masks& k, uint32_t w, uint32_t z0, uint32_t z1, uint32_t (&a)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v;  // (w >> 4 i & nibbles) | magic
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(w >> (4 * i)), "r"(k.nibbles), "r"(F16 ? k.f16 : k.bf16));
    a[i] = sub2<F16>(v, i & 1 ? z1 : z0);
  }
}

__device__ __forceinline__ uint4 load_codes(const uint4* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

__device__ __forceinline__ void store(void* y, int dtype, long long at, float v) {
  if (dtype == WAL_F32) static_cast<float*>(y)[at] = v;
  else if (dtype == WAL_F16) static_cast<__half*>(y)[at] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
}

// NT: tiles of eight tokens, GPC: groups in a chunk of 64 columns (1 or 2), F16: activations, STAGED: they are
// in shared memory
template <int NT, int GPC, bool F16, bool ZEROS, bool STAGED>
__global__ void __launch_bounds__(kThreads, 2) int4_gemv_kernel(const __grid_constant__ Int4Params p) {
  constexpr int LDR = 8 * NT + 1;
  __shared__ float red[kWarps][16][LDR];
  extern __shared__ __align__(16) uint8_t xs[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, q = lane & 3;
  const int own = kWarps / p.ks, groups = (p.tiles + own - 1) / own;  // row tiles of a group, and groups
  const int step = (int)gridDim.x, part = (int)blockIdx.x, chunks = p.chunks;
  const int wtile = warp / p.ks, kslice = warp % p.ks;
  const Masks masks = p.masks;

  struct Batch {
    uint4 w[kAhead];
    uint32_t s[kAhead][GPC];
    uint16_t z[kAhead][ZEROS ? GPC : 1];
  };
  // where a group's row tile of this warp begins: codes, scales and zeros of row r; a tile past the last one reads the last
  // one's (its rows are not written)
  struct Place {
    const uint4* w;
    const uint32_t* s;
    const uint16_t* z;
  };
  auto place = [&](int group) {
    const long long tile = min(group * own + wtile, p.tiles - 1);
    return Place{p.packed + tile * p.chunks * 32 + lane, p.scales + tile * p.groups * 8 + r, ZEROS ? p.zeros + tile * p.groups * 8 + r : nullptr};
  };
  auto fetch = [&](Batch& b, const Place& l, int c0) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int c = min(c0 + i * p.ks, chunks - 1);  // past the end: the last chunk's again, which nothing multiplies
      b.w[i] = load_codes(l.w + c * 32);
#pragma unroll
      for (int g = 0; g < GPC; ++g) {
        const int gi = GPC == 2 ? min(2 * c + g, p.groups - 1) : c >> p.per;
        // the half chunk behind K adds 0, not 0 times the last scale, which may be infinite
        b.s[i][g] = GPC == 2 && 2 * c + g >= p.groups ? 0u : __ldg(l.s + gi * 8);
        if (ZEROS) b.z[i][g] = __ldg(l.z + gi * 8);
      }
    }
  };

  Batch cur;
  Place here = place(part);
  wal_kv8::chain();  // the weights, too: the kernel before may be the one that packed or copied them
  fetch(cur, here, kslice);
  if (STAGED) {
    for (int row = warp; row < p.M; row += kWarps) {
      const uint4* from = reinterpret_cast<const uint4*>(p.x + row * p.ldx);
      for (int i = lane; i < chunks * 8; i += 32)  // zeros past K
        *reinterpret_cast<uint4*>(xs + row * p.stride + 16 * i) = i < p.K / 8 ? __ldg(from + i) : make_uint4(0u, 0u, 0u, 0u);
    }
    __syncthreads();
  }
  // this lane's activations of chunk 0, tokens r, r + 8, ..
  const uint8_t* const xl = STAGED ? xs + r * p.stride + 16 * q : reinterpret_cast<const uint8_t*>(p.x + r * p.ldx) + 16 * q;
  const long long xrows = STAGED ? 8ll * p.stride : 16 * p.ldx;  // bytes between them

  for (int group = part; group < groups; group += step) {
    float tot[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) tot[n][0] = tot[n][1] = tot[n][2] = tot[n][3] = 0.f;
    for (int c0 = kslice; c0 < chunks; c0 += kAhead * p.ks) {
      Batch next;
      const bool more = c0 + kAhead * p.ks < chunks;
      if (!more) here = place(min(group + step, groups - 1));
      fetch(next, here, more ? c0 + kAhead * p.ks : kslice);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int c = c0 + i * p.ks;
        if (c >= chunks) break;
        uint32_t xw[NT][2][4];  // columns 32 h + 8 q .. + 7 of token 8 n + r
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (8 * n + r < p.M && (STAGED || 64 * c + 32 * h + 8 * q < p.K)) {
              const uint4* from = reinterpret_cast<const uint4*>(xl + n * xrows + 128 * c + 64 * h);
              v = STAGED ? *from : __ldg(from);
            }
            xw[n][h][0] = v.x;
            xw[n][h][1] = v.y;
            xw[n][h][2] = v.z;
            xw[n][h][3] = v.w;
          }
        const uint32_t w[4] = {cur.w[i].x, cur.w[i].y, cur.w[i].z, cur.w[i].w};
        float acc[NT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int g = GPC == 2 ? h : 0;
          if (h == 0 || GPC == 2)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
          uint32_t z0 = F16 ? 0x64086408u : 0x43084308u, z1 = z0;
          if (ZEROS) {
            const uint32_t z = cur.z[i][g];
            z0 = (z & 0xffu) * 0x00010001u + magic<F16>();
            z1 = (z >> 8) * 0x00010001u + magic<F16>();
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t a[4];
            unpack<F16>(masks, w[2 * h + e], z0, z1, a);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma<F16>(acc[n], a, xw[n][h][2 * e], xw[n][h][2 * e + 1]);
          }
          if (h == 1 || GPC == 2) {
            const uint32_t sc = cur.s[i][g];
            const float s0 = __half2float(__ushort_as_half((unsigned short)(sc & 0xffffu)));
            const float s1 = __half2float(__ushort_as_half((unsigned short)(sc >> 16)));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              tot[n][0] = fmaf(s0, acc[n][0], tot[n][0]);
              tot[n][1] = fmaf(s0, acc[n][1], tot[n][1]);
              tot[n][2] = fmaf(s1, acc[n][2], tot[n][2]);
              tot[n][3] = fmaf(s1, acc[n][3], tot[n][3]);
            }
          }
        }
      }
      cur = next;
    }

    // the warps' sums
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[warp][r + 8 * (e >> 1)][8 * n + 2 * q + (e & 1)] = tot[n][e];
    __syncthreads();
    const int rows = own * 16;
    for (int i = tid; i < rows * p.M; i += kThreads) {
      const int row = i % rows, tok = i / rows;
      const long long n = (long long)group * rows + row;
      if (n >= p.N) continue;
      float v = 0.f;
      for (int k = 0; k < p.ks; ++k) v += red[(row >> 4) * p.ks + k][row & 15][tok];
      if (p.bias) v += __uint_as_float((uint32_t)p.bias[n] << 16);
      store(p.y, p.y_dtype, tok * p.ldy + n, v);
    }
    __syncthreads();
  }
}

// One word of packed codes per thread, and the first threads the scales and zeros.
__global__ void int4_pack_kernel(uint32_t* packed, uint32_t* scales, uint16_t* zeros, const uint8_t* codes, const uint16_t* s,
                                 const uint8_t* z, long long N, long long K, long long tiles, int chunks, int groups) {
  const long long words = tiles * chunks * 128, meta = tiles * groups * 8;
  const long long step = (long long)gridDim.x * blockDim.x;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < words; i += step) {
    const int w = (int)(i & 3), piece = (int)(i >> 2) & 31;
    const long long rest = i >> 7, c = rest % chunks, tile = rest / chunks;
    const long long row = tile * 16 + (piece >> 2), k = 64 * c + 32 * (w >> 1) + 8 * (piece & 3) + 4 * (w & 1);
    uint32_t v = 0;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const long long rr = row + 8 * (n & 1), kk = k + 2 * ((n >> 1) & 1) + (n >> 2);
      if (rr < N && kk < K) v |= (uint32_t)(codes[rr * K + kk] & 15) << (4 * n);
    }
    packed[i] = v;
  }
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < meta; i += step) {
    const int r = (int)(i & 7);
    const long long g = (i >> 3) % groups, row = (i >> 3) / groups * 16 + r;
    const bool lo = row < N, hi = row + 8 < N;
    scales[i] = (lo ? (uint32_t)s[row * groups + g] : 0u) | (hi ? (uint32_t)s[(row + 8) * groups + g] << 16 : 0u);
    if (zeros) zeros[i] = (uint16_t)((lo ? z[row * groups + g] & 15 : 0) | (hi ? (z[(row + 8) * groups + g] & 15) << 8 : 0));
  }
}

__global__ void int4_dequant_kernel(const uint32_t* packed, const uint16_t* scales, const uint8_t* zeros, void* w, long long ldw,
                                    int dtype, long long N, long long K, int chunks, int groups, int group_size) {
  const long long step = (long long)gridDim.x * blockDim.x;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < N * K; i += step) {
    const long long row = i / K, k = i % K, tile = row >> 4;
    const int rr = (int)(row & 15), c = (int)(k >> 6), j = (int)(k & 63);
    const int word = 2 * (j >> 5) + ((j >> 2) & 1), piece = 4 * (rr & 7) + ((j >> 3) & 3);
    const int nib = (rr >> 3) + 2 * ((j >> 1) & 1) + 4 * (j & 1);
    const uint32_t v = packed[((tile * chunks + c) * 32 + piece) * 4 + word];
    const long long m = ((tile * groups + k / group_size) * 8 + (rr & 7)) * 2 + (rr >> 3);
    const float z = zeros ? (float)zeros[m] : 8.f;
    store(w, dtype, row * ldw + k, ((float)((v >> (4 * nib)) & 15) - z) * __half2float(__ushort_as_half(scales[m])));
  }
}

int check_layer(const wal_int4_layer* l) {
  if (!l || !l->packed || !l->scales) return WAL_ERR_INVALID_ARGUMENT;
  size_t bytes, entries;
  const int st = wal_int4_packed_size(l->out_features, l->in_features, l->group_size, &bytes, &entries);
  if (st != WAL_OK) return st;
  if (((uintptr_t)l->packed & 15) || ((uintptr_t)l->scales & 15) || ((uintptr_t)l->zeros & 1)) return WAL_ERR_ALIGNMENT;
  return WAL_OK;
}

// What a CTA has for activations, two CTAs to an SM.
template <int NT>
constexpr int room() { return 227 * 1024 / 2 - 1024 - kWarps * 16 * (8 * NT + 1) * 4; }

template <int NT, int GPC, bool F16, bool ZEROS, bool STAGED>
int launch_one(const Int4Params& p, unsigned grid, cudaStream_t st) {
  auto kern = int4_gemv_kernel<NT, GPC, F16, ZEROS, STAGED>;
  if (STAGED) {
    static std::atomic<uint64_t> allowed{0};  // devices where the kernel may use its shared memory
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return WAL_ERR_CUDA;
    if (!(allowed.load(std::memory_order_relaxed) >> dev & 1)) {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, room<NT>()) != cudaSuccess) return WAL_ERR_CUDA;
      allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
  }
  return launch_chain(kern, dim3(grid), kThreads, STAGED ? p.M * p.stride : 0, st, p);
}

template <int NT, int GPC, bool ZEROS>
int launch_type(const Int4Params& p, unsigned grid, cudaStream_t st) {
  if ((long long)p.M * p.stride <= room<NT>())
    return p.f16 ? launch_one<NT, GPC, true, ZEROS, true>(p, grid, st) : launch_one<NT, GPC, false, ZEROS, true>(p, grid, st);
  return p.f16 ? launch_one<NT, GPC, true, ZEROS, false>(p, grid, st) : launch_one<NT, GPC, false, ZEROS, false>(p, grid, st);
}

template <int NT>
int launch(Int4Params p, int gpc, cudaStream_t st) {
  const int resident = 2 * sm_count();
  // the warps of a CTA share a tile or take several: what takes the fewest rounds of chunks (adding up costs about as much
  // as four)
  long long best = -1;
  unsigned grid = 1;
  for (int ks = 1; ks <= kWarps; ks *= 2) {
    const int own = kWarps / ks, groups = (p.tiles + own - 1) / own;
    const long long cost = (long long)((groups + resident - 1) / resident) * ((p.chunks + ks - 1) / ks + 4);
    if (best < 0 || cost < best) {
      best = cost;
      p.ks = ks;
      grid = (unsigned)(groups < resident ? groups : resident);
    }
  }
  if (gpc == 2) return p.zeros ? launch_type<NT, 2, true>(p, grid, st) : launch_type<NT, 2, false>(p, grid, st);
  return p.zeros ? launch_type<NT, 1, true>(p, grid, st) : launch_type<NT, 1, false>(p, grid, st);
}

}  // namespace

extern "C" {

int wal_int4_packed_size(int64_t out_features, int64_t in_features, int32_t group_size, size_t* packed_bytes, size_t* entries) {
  if (!packed_bytes || !entries) return WAL_ERR_INVALID_ARGUMENT;
  if (group_size != 32 && group_size != 64 && group_size != 128) return WAL_ERR_UNSUPPORTED;
  if (out_features <= 0 || in_features <= 0 || in_features % group_size) return WAL_ERR_SHAPE;
  if (out_features > (1 << 30) || in_features > (1 << 30)) return WAL_ERR_SHAPE;
  const size_t tiles = (size_t)((out_features + 15) / 16);
  *packed_bytes = tiles * (size_t)((in_features + 63) / 64) * 512;
  *entries = tiles * 16 * (size_t)(in_features / group_size);
  return WAL_OK;
}

int wal_int4_pack(const wal_int4_layer* l, const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, void* stream) {
  const int st = check_layer(l);
  if (st != WAL_OK) return st;
  if (!codes || !scales || !l->zeros != !zeros) return WAL_ERR_INVALID_ARGUMENT;
  int4_pack_kernel<<<sm_count() * 8, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<uint32_t*>(const_cast<void*>(l->packed)), reinterpret_cast<uint32_t*>(const_cast<uint16_t*>(l->scales)),
      reinterpret_cast<uint16_t*>(const_cast<uint8_t*>(l->zeros)), codes, scales, zeros, l->out_features, l->in_features,
      (l->out_features + 15) / 16, (int)((l->in_features + 63) / 64), (int)(l->in_features / l->group_size));
  return cudaGetLastError() == cudaSuccess ? WAL_OK : WAL_ERR_CUDA;
}

int wal_int4_dequant(const wal_int4_layer* l, void* w, int64_t ldw, int dtype, void* stream) {
  const int st = check_layer(l);
  if (st != WAL_OK) return st;
  if (!w) return WAL_ERR_INVALID_ARGUMENT;
  if (dtype != WAL_BF16 && dtype != WAL_F32 && dtype != WAL_F16) return WAL_ERR_UNSUPPORTED;
  if (ldw < l->in_features) return WAL_ERR_SHAPE;
  if ((uintptr_t)w & (dtype == WAL_F32 ? 3 : 1)) return WAL_ERR_ALIGNMENT;
  int4_dequant_kernel<<<sm_count() * 8, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint32_t*>(l->packed), l->scales, l->zeros, w, ldw, dtype, l->out_features, l->in_features,
      (int)((l->in_features + 63) / 64), (int)(l->in_features / l->group_size), l->group_size);
  return cudaGetLastError() == cudaSuccess ? WAL_OK : WAL_ERR_CUDA;
}

int wal_int4_gemv(const wal_int4_layer* l, const void* x, int x_dtype, int64_t M, int64_t ldx, void* y, int64_t ldy, int y_dtype,
                  void* stream) {
  const int st = check_layer(l);
  if (st != WAL_OK) return st;
  if (!x || !y) return WAL_ERR_INVALID_ARGUMENT;
  if (x_dtype != WAL_BF16 && x_dtype != WAL_F16) return WAL_ERR_UNSUPPORTED;
  if (y_dtype != WAL_BF16 && y_dtype != WAL_F32 && y_dtype != WAL_F16) return WAL_ERR_UNSUPPORTED;
  if (M <= 0 || M > 0x7fffffff || ldx < l->in_features || ldy < l->out_features) return WAL_ERR_SHAPE;
  const int ysize = y_dtype == WAL_F32 ? 4 : 2;
  if (((uintptr_t)x & 15) || (ldx % 8) || ((uintptr_t)y & (ysize - 1)) || (l->bias && ((uintptr_t)l->bias & 1))) return WAL_ERR_ALIGNMENT;
  Int4Params p = {};
  p.packed = static_cast<const uint4*>(l->packed);
  p.scales = reinterpret_cast<const uint32_t*>(l->scales);
  p.zeros = reinterpret_cast<const uint16_t*>(l->zeros);
  p.bias = l->bias;
  p.ldx = ldx;
  p.ldy = ldy;
  p.N = (int)l->out_features;
  p.K = (int)l->in_features;
  p.tiles = (p.N + 15) / 16;
  p.chunks = (p.K + 63) / 64;
  p.groups = p.K / l->group_size;
  p.per = l->group_size == 128 ? 1 : 0;
  p.y_dtype = y_dtype;
  p.f16 = x_dtype == WAL_F16;
  const int gpc = l->group_size == 32 ? 2 : 1;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  p.stride = p.chunks < 4096 ? 128 * p.chunks + 64 : 1 << 20;  // rows beyond are not staged anyway
  for (int64_t m0 = 0; m0 < M; m0 += 32) {
    p.M = (int)(M - m0 < 32 ? M - m0 : 32);
    p.x = static_cast<const uint16_t*>(x) + m0 * ldx;
    p.y = static_cast<uint8_t*>(y) + m0 * ldy * ysize;
    const int rc = p.M <= 8 ? launch<1>(p, gpc, s) : p.M <= 16 ? launch<2>(p, gpc, s) : launch<4>(p, gpc, s);
    if (rc != WAL_OK) return rc;
  }
  return WAL_OK;
}

}  // extern "C"
