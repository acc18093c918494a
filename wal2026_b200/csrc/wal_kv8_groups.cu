// Which rows of a page table share their first pages, and how far.
//
// Able rows (see the header) with the same page at position least - 1 are found
// by a hash table in shared memory that keeps the lowest row of each page; every
// row is then compared with that row, entry by entry, and the smallest agreement
// of a group's rows is what it shares.  One cluster: each CTA builds the same
// small table for itself, the comparisons (the only real reading) are dealt out to
// all warps, and the first CTA writes the groups down in order.
//
// On B200: 8 rows 5.9 us, 296 rows of up to 8700 positions in pages of 16 11.5 us (the
// comparisons read 0.3 MB): a chain of memory round trips and barriers.  Calls of more
// than 4096 table entries take the cluster, smaller ones a single CTA.
#include "wal_kv8.cuh"

#include <climits>
#include <cooperative_groups.h>

namespace {

namespace cg = cooperative_groups;
using namespace wal_kv8;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxRows = 4096;
constexpr int kSlots = 2 * kMaxRows;
constexpr int kCluster = 8;

struct GroupsParams {
  const int* table;
  long long ld_table;
  const int* lens;
  int rows, width, P, at;  // at: the entry that decides
  long long least;
  int slots;  // a power of two, at least 2 * rows
  int* groups;
};

struct Shared {
  int full[kMaxRows];    // whole pages of a row, -1 where it is not able
  int slot[kMaxRows];    // its place in the hash table; later its group's index and, at the leader, the start
  int common[kMaxRows];  // by leader: entries that all have in common
  int page[kSlots];
  int low[kSlots];       // lowest row of a page
  int size[kSlots];
  int wsum[kWarps];
};

__global__ void __launch_bounds__(kThreads) kv_pages_groups_kernel(const __grid_constant__ GroupsParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), ncta = (int)cl.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  chain();
  for (int i = tid; i < p.slots; i += kThreads) {
    s.page[i] = -1;
    s.low[i] = INT_MAX;
    s.size[i] = 0;
  }
  __syncthreads();
  for (int b = tid; b < p.rows; b += kThreads) {
    s.common[b] = INT_MAX;
    const long long n = min((long long)max(p.lens[b], 0), (long long)p.width * p.P - 1);
    int full = (int)(n / p.P);
    const int key = p.at < p.width ? p.table[b * p.ld_table + p.at] : -1;
    if (key < 0 || (long long)full * p.P / 32 * 32 < p.least) full = -1;
    s.full[b] = full;
    if (full < 0) continue;
    unsigned at = ((unsigned)key * 2654435761u) >> 16;
    for (int tries = 0; tries < p.slots; ++tries, ++at) {  // there are more slots than rows
      at &= (unsigned)(p.slots - 1);
      const int was = atomicCAS(&s.page[at], -1, key);
      if (was == -1 || was == key) break;
    }
    s.slot[b] = (int)at;
    atomicMin(&s.low[at], b);
    atomicAdd(&s.size[at], 1);
  }
  cl.sync();  // this CTA's table is there, and the first one's `common`
  for (int b = rank * kWarps + warp; b < p.rows; b += ncta * kWarps) {
    if (s.full[b] < 0) continue;
    const int lead = s.low[s.slot[b]];
    if (lead == b) continue;
    const int n = min(s.full[b], s.full[lead]);
    const int* mine = p.table + b * p.ld_table;
    const int* first = p.table + lead * p.ld_table;
    int same = n;
    for (int j = 0; j < n; j += 128) {
      bool differ = false;
      int at = INT_MAX;
#pragma unroll
      for (int u = 3; u >= 0; --u) {
        const int k = j + 32 * u + lane;
        if (k < n && __ldg(mine + k) != __ldg(first + k)) differ = true, at = k;
      }
      if (__any_sync(0xffffffffu, differ)) {
        same = __reduce_min_sync(0xffffffffu, at);
        break;
      }
    }
    if (lane == 0) atomicMin(cl.map_shared_rank(&s.common[lead], 0), same);
  }
  cl.sync();
  if (rank != 0) return;
  // groups by their lowest row: index and start of each, by a scan over the rows
  const int each = (p.rows + kThreads - 1) / kThreads, b0 = min(tid * each, p.rows), b1 = min(b0 + each, p.rows);
  auto positions = [&](int lead) { return (long long)min(s.common[lead], s.full[lead]) * p.P / 32 * 32; };
  auto leads = [&](int b) { return s.full[b] >= 0 && s.low[s.slot[b]] == b && s.size[s.slot[b]] > 1 && positions(b) >= p.least; };
  int count = 0, members = 0;  // at most 4096 each: one sum holds both
  for (int b = b0; b < b1; ++b)
    if (leads(b)) ++count, members += s.size[s.slot[b]];
  const int mine = count << 16 | members;
  int inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) s.wsum[warp] = inc;
  __syncthreads();
  int sum = inc - mine, total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) sum += s.wsum[w];
    total += s.wsum[w];
  }
  const int ngroups = total >> 16, nmembers = total & 0xffff;
  int* const order = p.groups;
  int* const begin = order + p.rows;
  int* const sizes = begin + p.rows;
  int* const shared = sizes + p.rows;
  for (int b = b0; b < b1; ++b) {
    if (!leads(b)) continue;
    const int sl = s.slot[b], n = s.size[sl];
    begin[sum >> 16] = sum & 0xffff;
    sizes[sum >> 16] = n;
    s.page[sl] = sum & 0xffff;  // where the next member goes
    sum += 1 << 16 | n;
  }
  for (int b = tid; b < p.rows; b += kThreads) {
    if (b >= ngroups) begin[b] = sizes[b] = 0;
    if (b >= nmembers) order[b] = -1;
    const int lead = s.full[b] >= 0 ? s.low[s.slot[b]] : b;
    shared[b] = leads(lead) ? (int)positions(lead) : 0;
  }
  __syncthreads();
  // members in rising order: one warp, 32 rows at a time
  if (warp == 0)
    for (int b = lane; b - lane < p.rows; b += 32) {
      const int lead = b < p.rows && s.full[b] >= 0 ? s.low[s.slot[b]] : -1;
      const bool in = lead >= 0 && leads(lead);
      const unsigned with = __match_any_sync(0xffffffffu, in ? lead : -1 - lane);
      int at = 0;
      if (in) at = s.page[s.slot[b]];
      __syncwarp();
      if (in) {
        order[at + __popc(with & ((1u << lane) - 1))] = b;
        if ((with >> lane) == 1u) s.page[s.slot[b]] = at + __popc(with);  // the last of them
      }
      __syncwarp();
    }
}

}  // namespace

extern "C" {

int wal_kv_pages_groups(const int32_t* table, int64_t ld_table, const int32_t* lens, int64_t rows, int64_t width,
                        int32_t page_size, int64_t least, int32_t* groups, void* stream) {
  if (!table || !lens || !groups) return WAL_ERR_INVALID_ARGUMENT;
  if (rows <= 0 || rows > kMaxRows || width <= 0 || ld_table < width || page_size <= 0 || least <= 0) return WAL_ERR_SHAPE;
  if (width >= 0x7fffffff || (width + 1) * (int64_t)page_size > (1LL << 31)) return WAL_ERR_SHAPE;
  GroupsParams p = {};
  p.table = table;
  p.ld_table = ld_table;
  p.lens = lens;
  p.rows = (int)rows;
  p.width = (int)width;
  p.P = page_size;
  p.at = (int)((least - 1) / page_size < width ? (least - 1) / page_size : width);
  p.least = least;
  p.slots = 64;
  while (p.slots < 2 * rows) p.slots *= 2;
  p.groups = groups;
  static std::atomic<uint64_t> allowed{0};  // devices where the kernel may use its shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return WAL_ERR_CUDA;
  if (!(allowed.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(kv_pages_groups_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared)) != cudaSuccess)
      return WAL_ERR_CUDA;
    allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  const int cluster = rows * width > 4096 ? kCluster : 1;
  return launch_chain(kv_pages_groups_kernel, dim3((unsigned)cluster), kThreads, (int)sizeof(Shared), static_cast<cudaStream_t>(stream),
                      p, cluster);
}

}  // extern "C"
