// Pages of the 8-bit KV cache: the tables of the next step (kept, forked,
// freed and new pages), compaction, and the copies both ask for.
//
//   kv_pages_assign_kernel   Counts the references that the kept prefixes make
//                            to each page, decides which partly filled last
//                            pages need a copy before they are written, and
//                            hands out free pages in rising order to the rows
//                            in rising order.  All counts are integers, so the
//                            result does not depend on the order of the atomics.
//   kv_pages_compact_kernel  Used pages beyond the live count move to the free
//                            pages below it, both in rising order.
//   kv_pages_copy_kernel     page src[i] -> dst[i] in every layer, K, V, scales.
//
// The first two are one cluster each, of one CTA for small pools and of eight or
// sixteen for large ones: what they do is a few dependent passes over a few hundred
// kilobytes, bound by the latency of the passes and of the barriers between, so
// rows are kept in shared memory and pages read eight at a time.  On B200: tables
// of 256 sequences with 65 k entries 15 us (96 us as one CTA, half of it atomics),
// of 64 forked rows 10 us, a compaction of 2055 pages 11 us.  The copy moves 266 MB
// of scattered 16 KB pieces in 50 us, 5.3 TB/s or 81% of a copy's rate; with CTAs
// that first list the valid pairs together it took 60 us.
#include "wal_kv8.cuh"

#include <cooperative_groups.h>

namespace {

namespace cg = cooperative_groups;
using namespace wal_kv8;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 16;  // at most

// Exclusive prefix sum over the CTA; *total gets the sum.  sm: kWarps ints.
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

// The same over the cluster, by rank; `box` (kCluster ints) is not used again by the kernel.  Ends with a cluster barrier.
__device__ __forceinline__ int cluster_scan(cg::cluster_group& cl, int v, int* sm, int* box, int* total) {
  const int rank = (int)cl.block_rank(), ncta = (int)cl.num_blocks();
  int mine;
  int at = block_scan(v, sm, &mine);
  if (threadIdx.x < ncta) cl.map_shared_rank(box, threadIdx.x)[rank] = mine;
  cl.sync();
  int sum = 0;
  for (int i = 0; i < ncta; ++i) {
    if (i < rank) at += box[i];
    sum += box[i];
  }
  *total = sum;
  return at;
}

// Chunks of kChunk entries of the rows of a table, one per warp at a time.
constexpr int kChunk = 512;

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
  extern __shared__ int begin[];  // [rows + 1] first wanted page of each row, [rows] kept pages, [rows] parents, bits of rows that copy
  __shared__ int scan[kWarps], box[kCluster];
  __shared__ unsigned long long lost;  // pages beyond the rows' width: up to 2^31 each
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), ncta = (int)cl.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gtid = rank * kThreads + tid, gthreads = ncta * kThreads, gwarp = rank * kWarps + warp, gwarps = ncta * kWarps;
  int* const have = begin + p.rows + 1;
  int* const parent = have + p.rows;  // minus one less the parent where the row writes into its last page
  unsigned* const copies = reinterpret_cast<unsigned*>(parent + p.rows);
  chain();
  // every CTA knows every row; a thread keeps its first row in registers
  Row first = {};
  int last_page = -1;  // that it will write
  for (int b = tid; b < p.rows; b += kThreads) {
    const Row r = load_row(p, b);
    have[b] = r.have;
    begin[b] = r.want;
    parent[b] = r.writes ? -1 - r.parent : r.parent;
    if (b == tid) first = r;
  }
  if (tid < p.rows) {
    if (first.writes) last_page = valid_page(__ldg(p.table + (long long)first.parent * p.ld_table + first.have - 1), p.pages);
  }
  if (tid == 0) lost = 0ull;
  for (int i = gtid; i < p.pages; i += gthreads) p.ref[i] = 0u;
  for (int i = tid; i < (p.rows + 31) / 32; i += kThreads) copies[i] = 0u;
  cl.sync();
  // kept entries and their references
  const int per_row = (p.width + kChunk - 1) / kChunk;
  for (long long u = gwarp; u < (long long)p.rows * per_row; u += gwarps) {
    const int b = (int)(u / per_row), j0 = (int)(u % per_row) * kChunk + lane;
    const int kept = have[b], want = begin[b], last = parent[b] < 0 ? kept - 1 : -1;
    const int* row = p.table + (long long)(parent[b] < 0 ? -1 - parent[b] : parent[b]) * p.ld_table;
    int e[kChunk / 32];
#pragma unroll
    for (int i = 0; i < kChunk / 32; ++i) {
      const int j = j0 + 32 * i;
      e[i] = j < kept ? valid_page(__ldg(row + j), p.pages) : -1;
    }
#pragma unroll
    for (int i = 0; i < kChunk / 32; ++i) {
      const int j = j0 + 32 * i;
      if (e[i] >= 0) atomicAdd(p.ref + e[i], j == last ? 0x10001u : 1u);
      if (j < p.width && (j < kept || j >= want)) p.out[(long long)b * p.ld_out + j] = e[i];
    }
  }
  cl.sync();
  // rows that write: sole owner, beside readers (a copy), or one of writers only (a copy unless it is the lowest)
  bool among = false;
  for (int b = tid; b < p.rows; b += kThreads) {
    Row r = first;
    int e = last_page;
    if (b >= kThreads) {
      r = load_row(p, b);
      e = r.writes ? valid_page(__ldg(p.table + (long long)r.parent * p.ld_table + r.have - 1), p.pages) : -1;
    }
    if (e >= 0) {
      const unsigned w = __ldcg(p.ref + e), total = w & 0xffffu, writers = w >> 16;
      if (total > 1) {
        atomicOr(copies + (b >> 5), 1u << (b & 31));
        among |= total == writers;
      }
    }
  }
  if (__syncthreads_or(among)) {  // the same in every CTA
    cl.sync();                    // nobody reads the counts any more
    for (int pass = 0; pass < 2; ++pass) {
      for (int b = tid; b < p.rows; b += kThreads) {
        if (!(copies[b >> 5] >> (b & 31) & 1u)) continue;
        int e = last_page;
        if (b >= kThreads) {
          const Row r = load_row(p, b);
          e = valid_page(__ldg(p.table + (long long)r.parent * p.ld_table + r.have - 1), p.pages);
        }
        const unsigned w = __ldcg(p.ref + e);
        if (pass == 0) {
          if ((w & kFlag) || (w & 0xffffu) == w >> 16) atomicMax(p.ref + e, kFlag | (kRowMask - (unsigned)b));
        } else if ((w & kFlag) && (w & kRowMask) == kRowMask - (unsigned)b) {
          atomicAnd(copies + (b >> 5), ~(1u << (b & 31)));
        }
      }
      cl.sync();
    }
  }
  // wanted pages of each row: its copy, then the new ones
  int base = 0;
  for (int b0 = 0; b0 < p.rows; b0 += kThreads) {
    const int b = b0 + tid;
    int n = 0, total;
    if (b < p.rows) {
      const Row r = b0 == 0 ? first : load_row(p, b);
      n = (int)(copies[b >> 5] >> (b & 31) & 1u) + r.want - r.have;
      const long long over = ((long long)r.keep + r.add + p.P - 1) / p.P - r.want;
      if (r.add && over > 0) atomicAdd(&lost, (unsigned long long)over);
    }
    const int at = block_scan(n, scan, &total);
    if (b < p.rows) begin[b] = base + at;
    base += total;
  }
  if (tid == 0) begin[p.rows] = base;
  // free pages in rising order to wanted ones in rising order; final counts.  Each thread has a run of pages.
  const int each = (p.pages + gthreads - 1) / gthreads, i0 = (int)min((long long)gtid * each, (long long)p.pages), i1 = min(i0 + each, p.pages);
  int mine = 0, found;
  for (int i = i0; i < i1; i += 8) {
    unsigned w[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) w[x] = i + x < i1 ? __ldcg(p.ref + i + x) : 1u;
#pragma unroll
    for (int x = 0; x < 8; ++x) mine += w[x] == 0u;
  }
  int k = cluster_scan(cl, mine, scan, box, &found);
  for (int i8 = i0; i8 < i1; i8 += 8) {
    unsigned words[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) words[x] = i8 + x < i1 ? __ldcg(p.ref + i8 + x) : 1u;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int i = i8 + x;
      const unsigned w = words[x];
      if (i >= i1) break;
      int count;
      if (w == 0u) {
        count = k < base;
        if (count) {
          int lo = 0, hi = p.rows - 1;  // the last row whose first wanted page is <= k
          while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (begin[mid] <= k) lo = mid;
            else hi = mid - 1;
          }
          const int s = k - begin[lo];
          const bool cow = copies[lo >> 5] >> (lo & 31) & 1u;
          if (cow && s == 0) p.dst[lo] = i;
          p.out[(long long)lo * p.ld_out + have[lo] + s - cow] = i;
        }
        ++k;
      } else if (w & kFlag) {
        count = 1;
      } else {
        const int t = w & 0xffffu, writers = w >> 16;
        count = t == writers ? 1 : t - writers;
      }
      p.ref[i] = (unsigned)count;
    }
  }
  // copies' sources, and what found no page
  for (int b = gtid; b < p.rows; b += gthreads) {
    const bool cow = copies[b >> 5] >> (b & 31) & 1u;
    int s = -1;
    if (cow && begin[b] < found) {
      s = p.table[(long long)(-1 - parent[b]) * p.ld_table + have[b] - 1];
    } else {
      p.dst[b] = -1;
    }
    p.src[b] = s;
    for (int x = max(begin[b], found); x < begin[b + 1]; ++x) p.out[(long long)b * p.ld_out + have[b] + x - begin[b] - cow] = -1;
  }
  if (rank == 0 && tid == 0) {
    p.info[0] = max(found - base, 0);
    p.info[1] = (int)min(lost + (unsigned long long)max(base - found, 0), 0x7fffffffull);
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
  __shared__ int scan[kWarps], box[3][kCluster];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), ncta = (int)cl.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gtid = rank * kThreads + tid, gthreads = ncta * kThreads, gwarp = rank * kWarps + warp, gwarps = ncta * kWarps;
  chain();
  for (int i = gtid; i < p.pages; i += gthreads) {
    p.remap[i] = -1;
    p.src[i] = -1;
    p.dst[i] = -1;
  }
  cl.sync();
  const int per_row = (p.width + kChunk - 1) / kChunk;
  for (long long u = gwarp; u < (long long)p.rows * per_row; u += gwarps) {
    const int b = (int)(u / per_row), j0 = (int)(u % per_row) * kChunk + lane;
    const int have = (min(max(p.lens[b], 0), p.width * p.P) + p.P - 1) / p.P;
    int e[kChunk / 32];
#pragma unroll
    for (int i = 0; i < kChunk / 32; ++i)
      e[i] = j0 + 32 * i < have ? valid_page(p.table[(long long)b * p.ld_table + j0 + 32 * i], p.pages) : -1;
#pragma unroll
    for (int i = 0; i < kChunk / 32; ++i)
      if (e[i] >= 0) p.remap[e[i]] = 0;
  }
  cl.sync();
  // each thread has a run of pages
  const int each = (p.pages + gthreads - 1) / gthreads, i0 = (int)min((long long)gtid * each, (long long)p.pages), i1 = min(i0 + each, p.pages);
  int mine = 0, live, movers, holes;
  for (int i = i0; i < i1; i += 8)
#pragma unroll
    for (int x = 0; x < 8; ++x) mine += i + x < i1 && __ldcg(p.remap + i + x) >= 0;
  const int used_before = cluster_scan(cl, mine, scan, box[0], &live);
  // holes below `live` and movers from there on follow from the used pages before a page
  int u = used_before, beyond = 0;
  if (i1 > live)
    for (int i = i0; i < i1; i += 8)
#pragma unroll
      for (int x = 0; x < 8; ++x) beyond += i + x >= live && i + x < i1 && __ldcg(p.remap + i + x) >= 0;
  int km = cluster_scan(cl, beyond, scan, box[1], &movers);
  for (int i8 = i0; i8 < i1; i8 += 8) {
    bool used[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) used[x] = i8 + x < i1 && __ldcg(p.remap + i8 + x) >= 0;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int i = i8 + x;
      if (i >= i1) break;
      if (used[x] && i >= live) p.src[km++] = i;
      if (!used[x] && i < live) p.dst[i - u] = i;
      if (used[x]) p.remap[i] = i;
      u += used[x];
    }
  }
  holes = movers;  // as many as there are movers
  cl.sync();
  for (int k = gtid; k < holes; k += gthreads) p.remap[__ldcg(p.src + k)] = __ldcg(p.dst + k);
  cl.sync();
  for (long long x = gwarp; x < (long long)p.rows * per_row; x += gwarps) {
    const int b = (int)(x / per_row), j0 = (int)(x % per_row) * kChunk + lane;
    const int have = (min(max(p.lens[b], 0), p.width * p.P) + p.P - 1) / p.P;
    int e[kChunk / 32];
#pragma unroll
    for (int i = 0; i < kChunk / 32; ++i)
      e[i] = j0 + 32 * i < have ? valid_page(p.table[(long long)b * p.ld_table + j0 + 32 * i], p.pages) : -1;
#pragma unroll
    for (int i = 0; i < kChunk / 32; ++i)
      if (e[i] >= 0) e[i] = __ldcg(p.remap + e[i]);
#pragma unroll
    for (int i = 0; i < kChunk / 32; ++i)
      if (j0 + 32 * i < p.width) p.out[(long long)b * p.ld_out + j0 + 32 * i] = e[i];
  }
  if (rank == 0 && tid == 0) {
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

// An item is 4 KB of one page and plane (layer, K or V) of one pair.  Warps take
// items a grid apart, so that those of a moved page go to as many warps and a
// list with few pairs in it (most of a compaction's is empty) still spreads;
// 32 items are looked up together, one per lane, and no warp waits for another.
constexpr int kCopyThreads = 128;
constexpr int kCopyCtasPerSm = 8;
constexpr int kItemVecs = 8;  // 16-byte pieces per lane
constexpr int kItemBytes = kItemVecs * 32 * 16;

__global__ void __launch_bounds__(kCopyThreads, kCopyCtasPerSm) kv_pages_copy_kernel(const __grid_constant__ CopyParams p) {
  const int lane = threadIdx.x & 31;
  const long long warps = (long long)gridDim.x * (kCopyThreads / 32), items = (long long)p.n * p.planes * p.segs;
  chain();
  for (long long it = (long long)blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5); it < items; it += 32 * warps) {
    const long long item = it + lane * warps;
    int s = -1, d = -1, plane = 0, seg = 0;
    if (item < items) {
      const long long i = item / (p.planes * p.segs);
      const int rest = (int)(item - i * (p.planes * p.segs));
      plane = rest / p.segs;
      seg = rest - plane * p.segs;
      s = valid_page(__ldg(p.src + i), p.pages);
      d = valid_page(__ldg(p.dst + i), p.pages);
    }
    unsigned todo = __ballot_sync(0xffffffffu, s >= 0 && d >= 0);
    while (todo) {
      const int l = __ffs(todo) - 1;
      todo &= todo - 1;
      const long long sp = __shfl_sync(0xffffffffu, s, l), dp = __shfl_sync(0xffffffffu, d, l);
      const int pl = __shfl_sync(0xffffffffu, plane, l), sg = __shfl_sync(0xffffffffu, seg, l);
      const long long off = (long long)sg * kItemBytes + lane * 16;
      uint8_t* const base = p.codes + pl * p.half_bytes + off;
      const int left = (int)min(p.page_bytes - off, (long long)kItemBytes);  // bytes from this lane's first piece on
      uint4 v[kItemVecs];
#pragma unroll
      for (int i = 0; i < kItemVecs; ++i)
        if (i * 512 < left) v[i] = __ldcs(reinterpret_cast<const uint4*>(base + sp * p.page_bytes + i * 512));
#pragma unroll
      for (int i = 0; i < kItemVecs; ++i)
        if (i * 512 < left) __stcs(reinterpret_cast<uint4*>(base + dp * p.page_bytes + i * 512), v[i]);
      if (sg == 0) {
        float* const sc = p.scales + pl * p.half_scales;
        for (int h = lane; h < p.hkv; h += 32) sc[dp * p.hkv + h] = sc[sp * p.hkv + h];
      }
    }
  }
}

// Dynamic shared memory of the assign kernel.
constexpr int assign_smem(int rows) { return (3 * rows + 1 + (rows + 31) / 32) * (int)sizeof(int); }
constexpr int kPlainSmem = 40 * 1024;  // a kernel may use this much without leave

// Lets the assign kernel use the shared memory of as many rows as it takes, once per
// device: an allowance that followed each call would be lowered by one thread between
// another's setting and launch.
bool allow_large_assign() {
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
  if (allowed.load(std::memory_order_relaxed) >> dev & 1) return true;
  if (cudaFuncSetAttribute(kv_pages_assign_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, assign_smem(kMaxRows)) != cudaSuccess)
    return false;
  allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  return true;
}

// CTAs of a table kernel's cluster, with the copy's time: one where each thread has
// at most one entry or page (36 pages of 6 sequences: 10.3 us with one or eight),
// eight for more (64 rows forked over 380 pages: 26.8 us with one, 25.2 with eight),
// and sixteen, where the device schedules clusters beyond the portable eight, when
// the entries' atomics and stores outweigh the barriers (256 sequences with 65 k
// entries: 24.8 us with eight, 16.5 with sixteen; 2055 pages with 1200 entries: 62 us either way).
// Whether sixteen fit is asked with as much shared memory as such calls use at most, apart
// for those that need leave for it: with it a CTA has an SM to itself.
template <typename Kern>
int table_cluster(Kern kern, int64_t entries, int64_t pages, int smem) {
  if (entries + pages <= kThreads) return 1;
  if (entries + pages <= 16 * kThreads) return 8;
  static std::atomic<int> known[2][kMaxDevices];  // 1: eight, 2: sixteen
  const bool large = smem > kPlainSmem;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 8;
  int can = known[large][dev].load(std::memory_order_relaxed);
  if (can == 0) {
    can = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kCluster);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)(large ? assign_smem(kMaxRows) : kPlainSmem);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kCluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
        cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) == cudaSuccess && clusters > 0)
      can = 2;
    (void)cudaGetLastError();  // a refusal is an answer
    known[large][dev].store(can, std::memory_order_relaxed);
  }
  return can == 2 ? kCluster : 8;
}

// Sizes whose indexes stay within 32 bits in the table kernels: strided loops over
// pages and chunks of entries run past their end by less than 2^30, and a row's
// tokens rounded up to pages are width * page_size + page_size - 1 at most.
bool table_fits(int64_t width, int64_t num_pages, int64_t page_size) {
  constexpr int64_t kMost = 1 << 30;
  return width <= kMost && num_pages <= kMost && width <= ((1LL << 31) - page_size) / page_size;
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
  if (rows > kMaxRows || rows_in > 0x7fffffff || !table_fits(width, num_pages, page_size)) return WAL_ERR_SHAPE;
  if (rows > 0x7fffffff / width) return WAL_ERR_SHAPE;  // wanted pages of all rows
  if (ld_table < width || ld_out < width) return WAL_ERR_SHAPE;
  AssignParams p = {table, ld_table, (int)rows_in, parent, keep, add, (int)rows, (int)width, (int)num_pages, page_size,
                    table_out, ld_out, reinterpret_cast<unsigned*>(ref_out), copy_src, copy_dst, info};
  const int smem = assign_smem((int)rows);
  if (smem > kPlainSmem && !allow_large_assign()) return WAL_ERR_CUDA;
  const int cluster = table_cluster(kv_pages_assign_kernel, rows * width, num_pages, smem);
  return launch_chain(kv_pages_assign_kernel, dim3((unsigned)cluster), kThreads, smem, static_cast<cudaStream_t>(stream), p, cluster);
}

int wal_kv_pages_compact(const int32_t* table, int64_t ld_table, const int32_t* lens, int64_t rows, int64_t width,
                         int64_t num_pages, int32_t page_size, int32_t* table_out, int64_t ld_out, int32_t* remap,
                         int32_t* move_src, int32_t* move_dst, int32_t* info, void* stream) {
  if (!table || !lens || !table_out || !remap || !move_src || !move_dst || !info) return WAL_ERR_INVALID_ARGUMENT;
  if (rows <= 0 || width <= 0 || num_pages <= 0 || page_size <= 0) return WAL_ERR_SHAPE;
  if (rows > 0x7fffffff || !table_fits(width, num_pages, page_size)) return WAL_ERR_SHAPE;
  if (ld_table < width || ld_out < width) return WAL_ERR_SHAPE;
  CompactParams p = {table, ld_table, lens, (int)rows, (int)width, (int)num_pages, page_size, table_out, ld_out, remap,
                     move_src, move_dst, info};
  const int cluster = table_cluster(kv_pages_compact_kernel, rows * width, num_pages, 0);
  return launch_chain(kv_pages_compact_kernel, dim3((unsigned)cluster), kThreads, 0, static_cast<cudaStream_t>(stream), p, cluster);
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
  if (2LL * cache->layers * ((p.page_bytes + kItemBytes - 1) / kItemBytes) > 0x7fffffff) return WAL_ERR_SHAPE;
  p.segs = (int)((p.page_bytes + kItemBytes - 1) / kItemBytes);
  p.src = src;
  p.dst = dst;
  p.n = (int)n;
  const long long items = (long long)n * p.planes * p.segs, ctas = (items + kCopyThreads / 32 - 1) / (kCopyThreads / 32);
  const long long most = (long long)kCopyCtasPerSm * sm_count();
  const dim3 grid((unsigned)(ctas < most ? ctas : most));
  return launch_chain(kv_pages_copy_kernel, grid, kCopyThreads, 0, static_cast<cudaStream_t>(stream), p);
}

}  // extern "C"
