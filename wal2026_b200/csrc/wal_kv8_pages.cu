// Pages of the 8-bit KV cache: the tables of the next step (kept, forked,
// freed and new pages), compaction, and the copies both ask for.
//
//   kv_pages_assign_kernel   one CTA.  Counts the references that the kept
//                            prefixes make to each page, decides which partly
//                            filled last pages need a copy before they are
//                            written, and hands out free pages in rising order
//                            to the rows in rising order.  All counts are
//                            integers, so the result does not depend on the
//                            order of the atomics.
//   kv_pages_compact_kernel  one CTA.  Used pages beyond the live count move to
//                            the free pages below it, both in rising order.
//   kv_pages_copy_kernel     page src[i] -> dst[i] in every layer, K, V, scales.
#include "wal_kv8.cuh"

namespace {

using namespace wal_kv8;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

// Exclusive prefix sum over the CTA; *total gets the sum.  sm: kWarps + 1 ints.
__device__ __forceinline__ int block_scan(int v, int* sm, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sm[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = sm[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    sm[lane] = s;
  }
  __syncthreads();
  *total = sm[kWarps - 1];
  return x - v + (warp ? sm[warp - 1] : 0);
}

struct AssignParams {
  const int* table;
  long long ld_table;
  int rows_in;
  const int* parent;
  const int* keep;
  const int* add;
  int rows, width, pages, P;
  int* out;
  long long ld_out;
  unsigned* ref;
  int* src;
  int* dst;
  int* info;
};

// A page's word while the kernel runs: references in the low 16 bits and, in
// the next 14, those of them that will write into the page (rows' partly
// filled last pages).  Pages whose references all write get kFlag plus the
// complement of the lowest such row.
constexpr unsigned kFlag = 0x40000000u, kRowMask = 0x3fffu;
constexpr int kMaxRows = 0x3fff;

struct Row {
  int parent, keep, add, have, want;  // tokens and pages, clamped to what a table row holds
  bool writes;
};

__device__ __forceinline__ Row load_row(const AssignParams& p, int b) {
  Row r;
  const int cap = p.width * p.P;
  r.parent = p.parent[b];
  r.keep = min(max(p.keep[b], 0), cap);
  if ((unsigned)r.parent >= (unsigned)p.rows_in) r.keep = 0;
  r.add = max(p.add[b], 0);
  r.have = (r.keep + p.P - 1) / p.P;
  const long long end = (long long)r.keep + r.add;
  r.want = r.add ? (int)min((end + p.P - 1) / p.P, (long long)p.width) : r.have;
  r.writes = r.add > 0 && r.keep % p.P != 0;
  return r;
}

__global__ void __launch_bounds__(kThreads) kv_pages_assign_kernel(const __grid_constant__ AssignParams p) {
  extern __shared__ int begin[];  // [rows + 1] first wanted page of each row
  __shared__ int scan[kWarps];
  __shared__ int lost;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) lost = 0;
  for (int i = tid; i < p.pages; i += kThreads) p.ref[i] = 0u;
  __syncthreads();
  // kept entries and their references
  for (int b = warp; b < p.rows; b += kWarps) {
    const Row r = load_row(p, b);
    for (int j = lane; j < p.width; j += 32) {
      int e = -1;
      if (j < r.have) {
        e = valid_page(p.table[(long long)r.parent * p.ld_table + j], p.pages);
        if (e >= 0) atomicAdd(p.ref + e, r.writes && j == r.have - 1 ? 0x10001u : 1u);
      }
      p.out[(long long)b * p.ld_out + j] = e;
    }
  }
  __syncthreads();
  // rows that write: sole owner, one of writers only, or beside readers
  for (int b = tid; b < p.rows; b += kThreads) {
    const Row r = load_row(p, b);
    const int e = r.writes ? p.out[(long long)b * p.ld_out + r.have - 1] : -1;
    int kind = 0;  // 1: copies, 2: copies unless it is the lowest writer
    if (e >= 0) {
      const unsigned w = __ldcg(p.ref + e), total = w & 0xffffu, writers = w >> 16;
      if (total > 1) kind = total == writers ? 2 : 1;
    }
    p.src[b] = e;
    p.dst[b] = kind;
  }
  __syncthreads();
  for (int b = tid; b < p.rows; b += kThreads)
    if (p.dst[b] == 2) atomicMax(p.ref + p.src[b], kFlag | (kRowMask - (unsigned)b));
  __syncthreads();
  // wanted pages of each row: its copy, then the new ones
  int base = 0;
  for (int b0 = 0; b0 < p.rows; b0 += kThreads) {
    const int b = b0 + tid;
    int n = 0, total;
    if (b < p.rows) {
      const Row r = load_row(p, b);
      bool cow = p.dst[b] == 1;
      if (p.dst[b] == 2) cow = (kRowMask - (__ldcg(p.ref + p.src[b]) & kRowMask)) != (unsigned)b;
      n = (cow ? 1 : 0) + r.want - r.have;
      if (!cow) p.src[b] = -1;
      p.dst[b] = -1;
      const long long over = ((long long)r.keep + r.add + p.P - 1) / p.P - r.want;
      if (r.add && over > 0) atomicAdd(&lost, (int)min(over, 0x3fffffffLL));
    }
    const int at = block_scan(n, scan, &total);
    if (b < p.rows) begin[b] = base + at;
    base += total;
    __syncthreads();
  }
  if (tid == 0) begin[p.rows] = base;
  __syncthreads();
  // free pages in rising order to wanted ones in rising order; final counts
  int given = 0, left = 0;
  for (int i0 = 0; i0 < p.pages; i0 += kThreads) {
    const int i = i0 + tid;
    unsigned w = 1u;
    if (i < p.pages) w = __ldcg(p.ref + i);
    int total;
    const int k = given + block_scan(w == 0u, scan, &total);
    if (i < p.pages) {
      int count;
      if (w == 0u) {
        count = k < base;
        left += !count;
        if (count) {
          int lo = 0, hi = p.rows - 1;  // the last row whose first wanted page is <= k
          while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (begin[mid] <= k) lo = mid;
            else hi = mid - 1;
          }
          const Row r = load_row(p, lo);
          int s = k - begin[lo];
          const bool cow = p.src[lo] >= 0;
          if (cow && s == 0) p.dst[lo] = i;
          const int j = cow ? r.have - 1 + s : r.have + s;
          p.out[(long long)lo * p.ld_out + j] = i;
        }
      } else if (w & kFlag) {
        count = 1;
      } else {
        const int t = w & 0xffffu, writers = w >> 16;
        count = t == writers ? 1 : t - writers;
      }
      p.ref[i] = (unsigned)count;
    }
    given += total;
    __syncthreads();
  }
  // what found no page
  if (given < base) {
    for (int b = tid; b < p.rows; b += kThreads)
      if (begin[b + 1] > given) {
        const Row r = load_row(p, b);
        const bool cow = p.src[b] >= 0;
        for (int k = max(begin[b], given); k < begin[b + 1]; ++k) {
          const int s = k - begin[b];
          p.out[(long long)b * p.ld_out + (cow ? r.have - 1 + s : r.have + s)] = -1;
          if (cow && s == 0) p.src[b] = -1;
        }
      }
  }
  int total;
  block_scan(left, scan, &total);
  if (tid == 0) {
    p.info[0] = total;
    p.info[1] = lost + (given < base ? base - given : 0);
  }
}

struct CompactParams {
  const int* table;
  long long ld_table;
  const int* lens;
  int rows, width, pages, P;
  int* out;
  long long ld_out;
  int* remap;
  int* src;
  int* dst;
  int* info;
};

__global__ void __launch_bounds__(kThreads) kv_pages_compact_kernel(const __grid_constant__ CompactParams p) {
  __shared__ int scan[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < p.pages; i += kThreads) {
    p.remap[i] = -1;
    p.src[i] = -1;
    p.dst[i] = -1;
  }
  __syncthreads();
  for (int b = warp; b < p.rows; b += kWarps) {
    const int have = (min(max(p.lens[b], 0), p.width * p.P) + p.P - 1) / p.P;
    for (int j = lane; j < have; j += 32) {
      const int e = valid_page(p.table[(long long)b * p.ld_table + j], p.pages);
      if (e >= 0) p.remap[e] = 0;
    }
  }
  __syncthreads();
  int mine = 0, live;
  for (int i = tid; i < p.pages; i += kThreads) mine += __ldcg(p.remap + i) >= 0;
  block_scan(mine, scan, &live);
  int movers = 0, holes = 0;
  for (int i0 = 0; i0 < p.pages; i0 += kThreads) {
    const int i = i0 + tid;
    const bool used = i < p.pages && __ldcg(p.remap + i) >= 0;
    const bool mover = used && i >= live, hole = i < p.pages && !used && i < live;
    int total;
    const int km = movers + block_scan(mover, scan, &total);
    movers += total;
    __syncthreads();
    const int kh = holes + block_scan(hole, scan, &total);
    holes += total;
    if (mover) p.src[km] = i;
    if (hole) p.dst[kh] = i;
    if (used) p.remap[i] = i;
    __syncthreads();
  }
  for (int k = tid; k < movers; k += kThreads) p.remap[p.src[k]] = p.dst[k];
  __syncthreads();
  for (int b = warp; b < p.rows; b += kWarps) {
    const int have = (min(max(p.lens[b], 0), p.width * p.P) + p.P - 1) / p.P;
    for (int j = lane; j < p.width; j += 32) {
      const int e = j < have ? valid_page(p.table[(long long)b * p.ld_table + j], p.pages) : -1;
      p.out[(long long)b * p.ld_out + j] = e >= 0 ? __ldcg(p.remap + e) : -1;
    }
  }
  if (tid == 0) {
    p.info[0] = live;
    p.info[1] = movers;
  }
}

struct CopyParams {
  uint8_t* codes;
  float* scales;
  long long page_bytes, half_bytes, half_scales;
  int hkv, pages, planes, segs;
  const int* src;
  const int* dst;
  int n;
};

constexpr int kCopyThreads = 256;
constexpr int kSegBytes = kCopyThreads * 16;  // bytes that one CTA copies of one page and plane

// grid.x: segments of a plane's page x planes (layer, K or V); grid.y: runs of 32 pairs.
__global__ void __launch_bounds__(kCopyThreads) kv_pages_copy_kernel(const __grid_constant__ CopyParams p) {
  const int seg = blockIdx.x % p.segs, plane = blockIdx.x / p.segs, lane = threadIdx.x & 31;
  for (int i0 = blockIdx.y * 32; i0 < p.n; i0 += gridDim.y * 32) {
    int s = -1, d = -1;
    if (i0 + lane < p.n) {
      s = valid_page(p.src[i0 + lane], p.pages);
      d = valid_page(p.dst[i0 + lane], p.pages);
    }
    unsigned todo = __ballot_sync(0xffffffffu, s >= 0 && d >= 0);
    while (todo) {
      const int l = __ffs(todo) - 1;
      todo &= todo - 1;
      const long long sp = __shfl_sync(0xffffffffu, s, l), dp = __shfl_sync(0xffffffffu, d, l);
      uint8_t* base = p.codes + plane * p.half_bytes;
      const long long off = (long long)seg * kSegBytes + threadIdx.x * 16;
      if (off < p.page_bytes)
        *reinterpret_cast<uint4*>(base + dp * p.page_bytes + off) = *reinterpret_cast<const uint4*>(base + sp * p.page_bytes + off);
      if (seg == 0) {
        float* sc = p.scales + plane * p.half_scales;
        for (int h = threadIdx.x; h < p.hkv; h += kCopyThreads) sc[dp * p.hkv + h] = sc[sp * p.hkv + h];
      }
    }
  }
}

}  // namespace

extern "C" {

int wal_kv_pages_assign(const int32_t* table, int64_t ld_table, int64_t rows_in, const int32_t* parent,
                        const int32_t* keep, const int32_t* add, int64_t rows, int64_t width, int64_t num_pages,
                        int32_t page_size, int32_t* table_out, int64_t ld_out, int32_t* ref_out, int32_t* copy_src,
                        int32_t* copy_dst, int32_t* info, void* stream) {
  if (!table || !parent || !keep || !add || !table_out || !ref_out || !copy_src || !copy_dst || !info)
    return WAL_ERR_INVALID_ARGUMENT;
  if (rows_in <= 0 || rows <= 0 || width <= 0 || num_pages <= 0 || page_size <= 0) return WAL_ERR_SHAPE;
  if (rows > kMaxRows || rows_in > 0x7fffffff || num_pages > 0x7fffffff - kThreads || width > 0x7fffffff / page_size)
    return WAL_ERR_SHAPE;
  if (ld_table < width || ld_out < width) return WAL_ERR_SHAPE;
  AssignParams p = {table, ld_table, (int)rows_in, parent, keep, add, (int)rows, (int)width, (int)num_pages, page_size,
                    table_out, ld_out, reinterpret_cast<unsigned*>(ref_out), copy_src, copy_dst, info};
  const int smem = ((int)rows + 1) * (int)sizeof(int);
  if (smem > 40 * 1024 && cudaFuncSetAttribute(kv_pages_assign_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return WAL_ERR_CUDA;
  kv_pages_assign_kernel<<<1, kThreads, smem, static_cast<cudaStream_t>(stream)>>>(p);
  return launch_status();
}

int wal_kv_pages_compact(const int32_t* table, int64_t ld_table, const int32_t* lens, int64_t rows, int64_t width,
                         int64_t num_pages, int32_t page_size, int32_t* table_out, int64_t ld_out, int32_t* remap,
                         int32_t* move_src, int32_t* move_dst, int32_t* info, void* stream) {
  if (!table || !lens || !table_out || !remap || !move_src || !move_dst || !info) return WAL_ERR_INVALID_ARGUMENT;
  if (rows <= 0 || width <= 0 || num_pages <= 0 || page_size <= 0) return WAL_ERR_SHAPE;
  if (rows > 0x7fffffff - kThreads || num_pages > 0x7fffffff - kThreads || width > 0x7fffffff / page_size) return WAL_ERR_SHAPE;
  if (ld_table < width || ld_out < width) return WAL_ERR_SHAPE;
  CompactParams p = {table, ld_table, lens, (int)rows, (int)width, (int)num_pages, page_size, table_out, ld_out, remap,
                     move_src, move_dst, info};
  kv_pages_compact_kernel<<<1, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return launch_status();
}

int wal_kv_pages_copy(const wal_kv8_cache* cache, const int32_t* src, const int32_t* dst, int64_t n, void* stream) {
  int st = check_cache(cache, 0);
  if (st != WAL_OK) return st;
  if (!src || !dst) return WAL_ERR_INVALID_ARGUMENT;
  if (n <= 0 || n > 0x7fffffff - 65536) return WAL_ERR_SHAPE;
  CopyParams p = {};
  p.codes = static_cast<uint8_t*>(cache->codes);
  p.scales = cache->scales;
  p.page_bytes = (long long)cache->kv_heads * cache->page_size * cache->head_dim;
  p.half_bytes = half_codes(*cache);
  p.half_scales = half_scales(*cache);
  p.hkv = cache->kv_heads;
  p.pages = (int)cache->num_pages;
  p.planes = 2 * cache->layers;
  p.segs = (int)((p.page_bytes + kSegBytes - 1) / kSegBytes);
  p.src = src;
  p.dst = dst;
  p.n = (int)n;
  const long long gx = (long long)p.planes * p.segs;
  if (gx > 0x7fffffff) return WAL_ERR_SHAPE;
  const long long runs = (n + 31) / 32;
  const dim3 grid((unsigned)gx, (unsigned)(runs < 1024 ? runs : 1024));
  kv_pages_copy_kernel<<<grid, kCopyThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return launch_status();
}

}  // extern "C"
