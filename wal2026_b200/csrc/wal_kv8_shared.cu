// Attention over the paged 8-bit KV cache for rows that share their first
// positions: what a group shares is read once for all of its rows.
//
// Two kernels.  The first one attends all query rows of a group (members x T tokens
// x G heads of a kv head, 128 to a tile) to the shared positions and leaves, for
// every row and head, (reference exponent, sum, weighted sum) in the workspace; the
// second one is the attention of wal_kv8_attn.cuh over each row's own positions,
// which joins the two.  Shared positions lie before every row's own, so
// there is no causal mask.
//
// The first kernel: a group of many samples has hundreds of rows per kv head, so
// its products run on the tensor cores by tcgen05 with both codes and weights as
// f16 (an int8 or e4m3 code is exact in f16).  Per 128 positions and 128 query rows,
// S = Q K^T and O += P V; Q is scaled by a power of two per row into f16's range, K
// codes and V codes stand in shared memory as f16 rows of positions (K-major for
// the first product, MN-major for the second: the same layout), S and O live in
// tensor memory, and P takes S's place there as the A operand of the second product.
//   warps 0-7   two slots of four warps, a query row per thread: maximum,
//               exponentials, sums, P, and the rescaling of O where the running
//               maximum has grown by 2^8; one slot's exponentials run beside the
//               other's products
//   warps 8-15  codes from global memory through registers to f16 in shared memory,
//               two stages; the next tile's loads are on their way meanwhile
//   warp 16     issues the products; warp 17 works out what the CTA has to do; warp 18
//               looks up pages and scales, some tiles ahead (loads that a loader
//               waits for hold up everything it asked for afterwards)
// A unit of up to 256 query rows of a kv head: more than 128 rows take a slot for
// each half, which share the converted codes; fewer give the slots alternate tiles.
// P is exp2(x - m + 7) times the block's V scale over a power of two that bounds
// the V scales so far: at most 2^15, so that f16 keeps weights down to 2^-32 of
// the largest; each is rounded by 2^-11 at most.  Maxima, sums and outputs are fp32.
//
// The position tiles of all units are cut into equal runs, one per SM.  Each run of
// a unit, and each slot that had some of its tiles, leaves a partial result; the
// second kernel reads those of a row in order, together with what the row has of its own,
// so the joining is spread over the whole GPU.  The second kernel starts while the
// first one runs and takes the SMs that it leaves.  Every wait is bounded by a deadline.
//
// Bounds, on B200.  64 rows over a document of 65700 positions (64 query, 8 kv heads
// of 128, int8, both kernels): 238 us, 573 TFLOP/s of the attention's own operations;
// its operations at the tensor cores' measured rate are 82 us, and reading the document
// once for every row would take 1300 us at a copy's rate.  A build with clocks in it spent
// about 6000 cycles on a tile of 128 positions and 256 rows, of which the tensor cores
// need 2048.  A slot's tile is a chain: its products and their commit 1400 cycles,
// maxima 600, exponentials 2400 (the special function units need 1024, twice where
// both slots are at it), P stored and its barrier 430.  Few rows: the same chain, and 16
// of a slot's 128 lanes at work; four samples of 2000 positions 20 us, where every row reading the
// prefix for itself takes 12.  Reading it once pays from about 100000 positions saved per call
// on (positions times members less one, 8 kv heads of 128); a call without groups costs 9 us more than
// kv8_attention.
// Steps of that case: first form 607 us; parts joined by the second kernel, 336; a
// warp that deals out the segments, 296; pages and scales by a warp of their own, 292;
// no spills in the loops and no clock read while polling, 250.  Not kept: sixteen softmax
// warps with half a row each (285 against 250), part of the exponentials by a polynomial
// and waits with a time hint (no change).
#include "wal_kv8_attn.cuh"

#include <type_traits>

namespace {

constexpr int kSlotWarps = 4, kSoftWarps = 8, kLoadWarps = 8;
constexpr int kPreThreads = 640;    // whole warpgroups; the last one issues the products and lays out the run
constexpr int kPreTile = 128;       // positions
constexpr int kPreCost = 1;         // what starting and ending a unit costs, in tiles of a slot
constexpr int kPreMin = 2;          // least cost of a run
constexpr int kMaxGroups = 2048;
constexpr int kMaxShared = 4096;    // rows of a call
constexpr unsigned long long kWaitNs = 2000000000ull;  // 2 s per wait, then give up
constexpr float kShift = 7.f;       // weights are 2^7 times exp2(x - m)
// Registers of the three kinds of warps: no more than the launch's 640 * 96 together.  (Nothing may spill in the loops:
// with this much shared memory taken, two spilled words in three come back from L2.)
constexpr int kSoftRegs = 120, kLoadRegs = 80, kIssueRegs = 80;
static_assert(256 * kSoftRegs + 256 * kLoadRegs + 128 * kIssueRegs <= kPreThreads * 96, "registers of the launch");

struct PreParams {
  const uint16_t* q;
  long long ld_q;
  LayerView kv;
  int B, T, hq, hkv, G, P, pages, max_pages;
  const int* table;
  long long ld_table;
  const int* new_lens;
  const int* groups;  // [4][B]
  float qscale;
  PrefixParts parts;
  int* status;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint64_t globaltimer() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(ok)
               : "r"(bar), "r"(parity)
               : "memory");
  return ok != 0;
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

// Operand in shared memory, rows of 64 f16 (128 bytes, 16-byte pieces xor row % 8), eight rows 1024 bytes apart.
// K-major: rows are the other dimension.  MN-major: rows are k, the next 64 columns `lead` bytes further.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)((lead >> 4) & 0x3fff) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
// fp32 = f16 x f16, M = 128
__host__ __device__ constexpr uint32_t instruction(int n, bool b_mn_major) {
  return (1u << 4) | (b_mn_major ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
               "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
               "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr)
      : "memory");
}
// The registers pass through the wait, so that no use of them comes before it.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};\n" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(addr)
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n" ::"r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
      "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(addr)
      : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Two fp32 numbers at once.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Codes pass once: they leave L1 to what little else is there.
__device__ __forceinline__ uint4 load_codes(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// Four codes of a word, in order, as two registers of f16.
template <int KIND>
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t& a, uint32_t& b) {
  if (KIND == WAL_KV_INT8) {
    const uint32_t u = w ^ 0x80808080u;  // code + 128 as the low byte of 1024 + it
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(a) : "r"(__byte_perm(u, 0x64646464u, 0x4140)), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(b) : "r"(__byte_perm(u, 0x64646464u, 0x4342)), "r"(0x64806480u));
  } else {
    asm("{.reg .b16 lo, hi;\n mov.b32 {lo, hi}, %2;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n cvt.rn.f16x2.e4m3x2 %1, hi;\n}"
        : "=r"(a), "=r"(b)
        : "r"(w));
  }
}

template <int HD>
struct PreShape {
  static constexpr int kHalf = kPreTile * 128;        // 64 columns of 128 rows
  static constexpr int kOperand = kHalf * (HD / 64);  // Q of a slot, a stage of K, a stage of V
  static constexpr int kStages = 2;
  static constexpr int kSmem = 1024 + kOperand * (2 + 2 * kStages);
  // tensor memory columns of slot s
  __host__ __device__ static constexpr int s_at(int s) { return 128 * s; }
  __host__ __device__ static constexpr int o_at(int s) { return 256 + HD * s; }
  // P: over the first half of the scores, which the next first product (of the same shape as the second one, and so
  // after it) overwrites; in a place of its own where there is room
  __host__ __device__ static constexpr int p_at(int s) { return HD == 128 ? 128 * s : 384 + 64 * s; }
};

// What one CTA takes of a unit.
struct PreSegment {
  int begin;         // of the members in groups[0]; negative: there is no more
  int positions;     // shared
  int rows0, rows;   // first query row of the unit, and how many there are (up to 256)
  int kvh;
  int tile0, tile1;
  int both;          // more than 128 rows: a slot for each half
};
constexpr int kSegRing = 4;
constexpr int kAhead = 8;

// Scales of a block of 16 positions: K scale, log2 and reciprocal of the V scale.
struct Block {
  float k, lv, rv, unused;
};

struct PreState {
  unsigned prefix[kMaxGroups + 1];   // cost before each group
  int positions[kMaxGroups];         // that it shares
  PreSegment seg[kSegRing];          // written by the scheduler, read by the others
  // of a tile, for kAhead tiles
  Block side[kAhead][8];
  int page[kAhead][8];               // of its blocks of 16 positions
  unsigned have[kAhead];             // blocks that have a page
  int top[kAhead];                   // exponent of a power of two that bounds a tile's V scales
  long long wsum[kPreThreads / 32];
  unsigned long long bars[40];
  uint32_t tmem;
  int abort;
};

constexpr float kTinyScale = 7.888609052210118e-31f;  // 2^-100: V scales count as no less
constexpr float kFarLog = -96.f, kFar = 7.922816251426434e28f;  // nor as less than 2^-96 of the largest

// The i-th group, or nothing where its numbers do not fit the call.
__device__ __forceinline__ bool group_of(const PreParams& p, int i, int& begin, int& size, int& positions) {
  begin = p.groups[p.B + i];
  size = p.groups[2 * p.B + i];
  if (size <= 0 || begin < 0 || begin >= p.B || size > p.B - begin) return false;
  const int lead = p.groups[begin];
  if ((unsigned)lead >= (unsigned)p.B) return false;
  positions = (int)min((long long)p.groups[3 * p.B + lead], (long long)p.max_pages * p.P) & ~31;
  return positions > 0;
}

// Number of the i-th group's first unit; the groups before it have fewer units than that.
__device__ __forceinline__ int unit_base(const PreParams& p, int i, int begin) {
  return (int)(p.hkv * (i + (long long)begin * p.T * p.G / kUnitRows));
}

template <int HD, int KIND>
__global__ void __launch_bounds__(kPreThreads, 1) kv8_prefix_kernel(const __grid_constant__ PreParams p) {
  using S = PreShape<HD>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ PreState st;
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  const uint32_t q_sm = base, k_sm = q_sm + 2 * S::kOperand, v_sm = k_sm + S::kStages * S::kOperand;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t bars = smem_u32(st.bars);
  // by stage: kfull, vfull, kfree, vfree; by slot: sfull, pfull, qfull; by tile: sidefull, sidefree
  const uint32_t kfull = bars, vfull = bars + 16, kfree = bars + 32, vfree = bars + 48, sfull = bars + 64, pfull = bars + 80;
  const uint32_t qfull = bars + 96, oend = bars + 112, drained = bars + 120, segfull = bars + 128, segfree = bars + 160;
  const uint32_t sidefull = bars + 192, sidefree = bars + 256;
  volatile int* const abort = &st.abort;

  if (tid == 0) {
    st.abort = 0;
    for (int s = 0; s < 2; ++s) {
      mbar_init(kfull + 8 * s, kLoadWarps);
      mbar_init(vfull + 8 * s, kLoadWarps);
      mbar_init(kfree + 8 * s, 1);
      mbar_init(vfree + 8 * s, 1);
      mbar_init(sfull + 8 * s, 1);
      mbar_init(pfull + 8 * s, kSlotWarps);
      mbar_init(qfull + 8 * s, kSlotWarps);
    }
    mbar_init(oend, 1);
    mbar_init(drained, 1);
    for (int s = 0; s < kAhead; ++s) {
      mbar_init(sidefull + 8 * s, 1);
      mbar_init(sidefree + 8 * s, 1);
    }
    for (int s = 0; s < kSegRing; ++s) {
      mbar_init(segfull + 8 * s, 1);
      mbar_init(segfree + 8 * s, kSoftWarps + kLoadWarps + 2);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&st.tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  chain();
  // cost of the groups and their running sum
  const int ng = min(p.B / 2, kMaxGroups);
  {
    const int each = (ng + kPreThreads - 1) / kPreThreads, i0 = min(tid * each, ng), i1 = min(i0 + each, ng);
    auto unit_rows = [&](int size) { return (long long)size * p.T * p.G; };
    auto cost = [&](int i) -> long long {
      int begin, size, positions;
      if (!group_of(p, i, begin, size, positions)) return 0;
      st.positions[i] = positions;
      const long long rows = unit_rows(size), pairs = rows / kUnitRows, rest = rows % kUnitRows;
      const int tiles = (positions + kPreTile - 1) / kPreTile;
      return p.hkv * (pairs * (2 * tiles + kPreCost) + (rest ? (rest > kSlotRows ? 2 : 1) * tiles + kPreCost : 0));
    };
    long long mine = 0;
    for (int i = i0; i < i1; ++i) {
      const long long c = cost(i);
      st.prefix[i] = (unsigned)c;
      mine += c;
    }
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) st.wsum[warp] = inc;
    __syncthreads();
    long long sum = inc - mine;
    for (int w = 0; w < warp; ++w) sum += st.wsum[w];
    for (int i = i0; i < i1; ++i) {
      const unsigned c = st.prefix[i];
      st.prefix[i] = (unsigned)sum;
      sum += c;
    }
    // groups of a table fit 32 bits (the host has seen to it); of others that do not, nothing is done
    if (tid == kPreThreads - 1) st.prefix[ng] = sum < (1ll << 31) ? (unsigned)sum : 0u;
    // where the second kernel finds a row's group
    for (int i = blockIdx.x; i < ng; i += gridDim.x) {
      int begin, size, positions;
      if (!group_of(p, i, begin, size, positions)) continue;
      const long long tg = (long long)p.T * p.G;
      const int heads = (int)((size * tg + kUnitRows - 1) / kUnitRows);  // units of a kv head
      for (int j = tid; j < size; j += kPreThreads) {
        const int b = p.groups[begin + j];
        if ((unsigned)b < (unsigned)p.B) p.parts.rows[b] = make_int4(unit_base(p, i, begin), j, heads, 0);
      }
    }
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = st.tmem;
  auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
    uint64_t t0 = 0;
    while (true) {
      // a warp that spins takes issue slots from those that work, so the clock is looked at now and then
#pragma unroll 1
      for (int i = 0; i < 64; ++i)
        if (mbar_try(bar, parity)) return true;
      if (*abort) return false;
      const uint64_t now = globaltimer();
      if (t0 == 0) t0 = now;
      if (now - t0 > kWaitNs) {
        *abort = 1;
        if (p.status) *p.status = 1;
        return false;
      }
    }
  };
  // the same for all lanes of a warp
  auto warp_wait = [&](uint32_t bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, wait(bar, parity)); };

  if (warp < kSoftWarps) {
    // ------------------------------------------------ softmax: thread = query row of a slot
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    const int slot = warp / kSlotWarps, srow = tid % kSlotRows;
    const uint32_t lanes = tmem + ((uint32_t)((warp % 4) * 32) << 16);
    const uint32_t s_at = lanes + S::s_at(slot), o_at = lanes + S::o_at(slot), p_at = lanes + S::p_at(slot);
    unsigned mine = 0, seen = 0;  // tiles of this slot, and of all
    bool ok = true;
    for (unsigned seg = 0; ok; ++seg) {
      if (!(ok = warp_wait(segfull + 8 * (seg % kSegRing), (seg / kSegRing) & 1))) break;
      const PreSegment& sg = st.seg[seg % kSegRing];
      if (sg.begin < 0) break;
      const int both = sg.both, r = both ? slot * kSlotRows + srow : srow;
      // this thread's query row, if there is one
      bool real = r < sg.rows;
      unsigned token = 0, head = 0;  // b * T + t, and the query head
      if (real) {
        const unsigned row = (unsigned)(sg.rows0 + r), one = (unsigned)(p.T * p.G), member = row / one, in = row - member * one;
        const unsigned t = in / (unsigned)p.G;
        const int b = p.groups[sg.begin + (int)member];
        real = (unsigned)b < (unsigned)p.B && (!p.new_lens || (int)t < p.new_lens[b]);
        if (real) {
          token = (unsigned)(b * p.T) + t;
          head = (unsigned)(sg.kvh * p.G) + in - t * (unsigned)p.G;
        }
      }
      // q, scaled into f16's range; where both slots work on the same rows the first one writes it
      float unscale;
      {
        const uint4* src = reinterpret_cast<const uint4*>(p.q + (long long)token * p.ld_q + (long long)head * HD);
        // read twice, a few pieces at a time: all of the row in registers would push what the loop below needs out of them
        float mx = 0.f;
#pragma unroll 1
        for (int i0 = 0; i0 < HD / 8; i0 += 4) {
          uint4 w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = real ? __ldg(src + i0 + i) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = max3(mx, fabsf(bf16_lo(u[e])), fabsf(bf16_hi(u[e])));
          }
        }
        const int e2 = min(max(14 + 127 - (int)(__float_as_uint(mx) >> 23), -112), 126);
        // q takes the scale's sign, so that the largest product stays the largest score
        const float up = copysignf(__uint_as_float((uint32_t)(e2 + 127) << 23), p.qscale);
        unscale = fabsf(p.qscale) * __uint_as_float((uint32_t)(127 - e2) << 23);
        if (slot == 0 || both) {
#pragma unroll 1
          for (int i0 = 0; i0 < HD / 8; i0 += 4) {
            uint4 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = real ? __ldg(src + i0 + i) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
              uint32_t h[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) h[e] = pack_f16(bf16_lo(u[e]) * up, bf16_hi(u[e]) * up);
              const int k = i0 + i;
              const uint32_t dst = q_sm + slot * S::kOperand + (k >> 3) * S::kHalf + srow * 128 + (((k & 7) ^ (srow & 7)) << 4);
              asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
            }
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(qfull + 8 * slot);
      const bool some = __any_sync(0xffffffffu, real);  // a warp without rows only keeps step
      float m = -INFINITY, l = 0.f;
      int eref = -200;  // exponent of what V scales are taken relative to
      bool first = true;
      const int n = sg.tile1 - sg.tile0;
      for (int i = both ? 0 : slot; i < n; i += both ? 1 : 2, ++mine) {
        const unsigned at = seen + i, entry = at % kAhead;
        if (!(ok = warp_wait(sfull + 8 * slot, mine & 1))) break;
        if (!(ok = warp_wait(sidefull + 8 * entry, (at / kAhead) & 1))) break;
        tc_after();
        if (some) {
          const Block* side = st.side[entry];
          const unsigned have = st.have[entry];
          const int left = sg.positions - (sg.tile0 + i) * kPreTile, etop = st.top[entry];  // left: a multiple of 32
          const bool full = have == 0xffu && left >= kPreTile;
          // a block of 16 positions at a time, the next one on its way, from the last to the first and back: P takes the
          // place of scores that are in registers or done with
          uint32_t xa[16], xb[16];
          float mn = -INFINITY;
          auto largest = [&](const uint32_t (&x)[16], int k) {
            float t0 = max3(__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]));
            float t1 = max3(__uint_as_float(x[3]), __uint_as_float(x[4]), __uint_as_float(x[5]));
#pragma unroll
            for (int e = 6; e < 14; e += 4) {
              t0 = max3(t0, __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
              t1 = max3(t1, __uint_as_float(x[e + 2]), __uint_as_float(x[e + 3]));
            }
            t0 = max3(t0, __uint_as_float(x[14]), __uint_as_float(x[15]));
            const float top = fmaxf(t0, t1) * (unscale * side[k].k);
            mn = full || (16 * k < left && ((have >> k) & 1)) ? fmaxf(mn, top) : mn;
          };
          tmem_ld16(s_at + 112, xa);
#pragma unroll
          for (int k = 7; k > 0; k -= 2) {
            tmem_ld_wait(xa);
            tmem_ld16(s_at + 16 * (k - 1), xb);
            largest(xa, k);
            tmem_ld_wait(xb);
            tmem_ld16(s_at + 16 * (k > 1 ? k - 2 : 1), xa);  // after the first block the second one again
            largest(xb, k - 1);
          }
          if (__any_sync(0xffffffffu, first || mn > m + kSlack || etop > eref)) {
            const float top = fmaxf(m, mn);
            const float al = top == -INFINITY ? 0.f : ex2(m - top);
            const float f = al * (etop > eref ? ex2((float)max(eref - etop, -126)) : 1.f);
            eref = max(eref, etop);
            m = top;
            l *= al;
            if (!first) {  // the products before have finished: this tile's S came after them
#pragma unroll
              for (int c = 0; c < HD / 16; ++c) {
                uint32_t o[16];
                tmem_ld16(o_at + 16 * c, o);
                tmem_ld_wait(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st16(o_at + 16 * c, o);
              }
            }
          }
          first = false;
          const float off = m == -INFINITY ? 0.f : kShift - m, up = __uint_as_float((uint32_t)(max(eref, -126) + 127) << 23);
          // S * f + off in one rounding, whose reference is -off itself.  Where m is so large that its own rounding shows in
          // the exponent, the product is rounded as the maximum's was; that form also leaves out blocks.
          auto weights = [&](auto plain, const uint32_t (&x)[16], int k) {
            uint32_t w[8];
            const Block bl = side[k];
            const float f = unscale * bl.k, lv = fmaxf(bl.lv - (float)eref, kFarLog);
            float sum = 0.f;
            if (plain.value) {
              const uint64_t f2 = pair2(f, f), o2 = pair2(off + lv, off + lv);
              uint64_t s2 = 0ull;
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                float a, d;
                split2(fma2(pair2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), f2, o2), a, d);
                a = ex2(a);
                d = ex2(d);
                s2 = add2(s2, pair2(a, d));
                w[e / 2] = pack_f16(a, d);
              }
              float a, d;
              split2(s2, a, d);
              sum = a + d;
            } else {
              const bool in = 16 * k < left && ((have >> k) & 1);
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                const float a = in ? ex2(__fadd_rn(__fadd_rn(__fmul_rn(__uint_as_float(x[e]), f), off), lv)) : 0.f;
                const float d = in ? ex2(__fadd_rn(__fadd_rn(__fmul_rn(__uint_as_float(x[e + 1]), f), off), lv)) : 0.f;
                sum += a + d;
                w[e / 2] = pack_f16(a, d);
              }
            }
            l = fmaf(sum, fminf(bl.rv * up, kFar), l);
            tmem_st8(p_at + 8 * k, w);
          };
          auto second = [&](auto plain) {
            weights(plain, xb, 0);
#pragma unroll
            for (int k = 1; k < 8; k += 2) {
              tmem_ld_wait(xa);
              if (k < 7) tmem_ld16(s_at + 16 * (k + 1), xb);
              weights(plain, xa, k);
              if (k < 7) {
                tmem_ld_wait(xb);
                tmem_ld16(s_at + 16 * (k + 2), xa);
                weights(plain, xb, k + 1);
              }
            }
          };
          if (__any_sync(0xffffffffu, !full || fabsf(off) > 65536.f)) second(std::false_type{});
          else second(std::true_type{});
          tmem_st_wait();
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(pfull + 8 * slot);
      }
      if (!ok) break;
      seen += n;
      // the unit's sums: O after the segment's last product
      if (!(ok = warp_wait(oend, seg & 1))) break;
      tc_after();
      if (some) {
        const float up = __uint_as_float((uint32_t)(max(eref, -126) + 127) << 23);
        const bool lead = sg.tile0 == 0;
        // the unit's first run: by row; a later one, which leads this CTA's run: by CTA
        const long long part = lead ? 2 * ((long long)token * p.hq + head) + (both ? 0 : slot) : (2ll * blockIdx.x + slot) * kSlotRows + srow;
        float* dst = (lead ? p.parts.first : p.parts.later) + part * HD;
        const bool any = !first;  // this slot had a tile
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          if (!any) break;
          uint32_t x[32];
          tmem_ld32(o_at + 32 * c, x);
          tmem_ld_wait(x);
          if (real)
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              __stcg(reinterpret_cast<float4*>(dst + 32 * c + e),
                     make_float4(__uint_as_float(x[e]) * up, __uint_as_float(x[e + 1]) * up, __uint_as_float(x[e + 2]) * up,
                                 __uint_as_float(x[e + 3]) * up));
        }
        if (real) (lead ? p.parts.first_stats : p.parts.later_stats)[part] = make_float2(m == -INFINITY ? 0.f : -(kShift - m), l);
      }
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(segfree + 8 * (seg % kSegRing));
    }
  } else if (warp < kSoftWarps + kLoadWarps) {
    // ------------------------------------------------ codes to f16
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
    // a thread has 16-byte pieces 4 h + (ct % 4) of rows ct / 4 and ct / 4 + 64: the stores of eight lanes meet no bank twice
    constexpr int HALVES = HD / 64, ROWS = 2;
    const int ct = tid - 32 * kSoftWarps, piece = ct & 3, row = ct >> 2;
    const long long page_codes = (long long)p.hkv * p.P * HD;
    const uint32_t swz = (uint32_t)(row * 128 + (((2 * piece) ^ (row & 7)) << 4));  // the odd piece is 16 bytes off by xor
    unsigned seen = 0, uses0 = 0, uses1 = 0;  // tiles; uses of the stages
    bool ok = true;
    for (unsigned seg = 0; ok; ++seg) {
      if (!(ok = warp_wait(segfull + 8 * (seg % kSegRing), (seg / kSegRing) & 1))) break;
      const PreSegment& sg = st.seg[seg % kSegRing];
      if (sg.begin < 0) break;
      const int n = sg.tile1 - sg.tile0;
      const long long off = (long long)sg.kvh * p.P * HD + (row & (p.P - 1)) * HD + piece * 16;  // 64 is a whole number of pages
      const uint8_t *kbase = p.kv.k + off, *vbase = p.kv.v + off;
      __syncwarp();
      if (lane == 0) mbar_arrive(segfree + 8 * (seg % kSegRing));  // all of it has been read
      uint4 kd[ROWS][HALVES], vd[ROWS][HALVES];
      auto fetch = [&](const uint8_t* from, uint4 (&d)[ROWS][HALVES], unsigned at) {
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
          const int page = st.page[at % kAhead][row / 16 + 4 * j];
          const uint8_t* src = from + max(page, 0) * page_codes;
#pragma unroll
          for (int h = 0; h < HALVES; ++h) d[j][h] = page >= 0 ? load_codes(src + 64 * h) : make_uint4(0u, 0u, 0u, 0u);
        }
      };
      auto put = [&](uint32_t stage_sm, const uint4 (&d)[ROWS][HALVES]) {
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            uint32_t w[8];
            codes_f16<KIND>(d[j][h].x, w[0], w[1]);
            codes_f16<KIND>(d[j][h].y, w[2], w[3]);
            codes_f16<KIND>(d[j][h].z, w[4], w[5]);
            codes_f16<KIND>(d[j][h].w, w[6], w[7]);
            const uint32_t dst = stage_sm + h * S::kHalf + j * 64 * 128;
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + swz), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + (swz ^ 16u)), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
          }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      };
      if (!(ok = warp_wait(sidefull + 8 * (seen % kAhead), (seen / kAhead) & 1))) break;
      fetch(kbase, kd, seen);
      fetch(vbase, vd, seen);
      for (int i = 0; i < n; ++i) {
        const unsigned stage = i & 1, use = stage ? uses1++ : uses0++;
        const bool more = i + 1 < n;
        ++seen;
        if (use && !(ok = warp_wait(kfree + 8 * stage, (use - 1) & 1))) break;
        put(k_sm + stage * S::kOperand, kd);
        __syncwarp();
        if (lane == 0) mbar_arrive(kfull + 8 * stage);
        if (more) {
          if (!(ok = warp_wait(sidefull + 8 * (seen % kAhead), (seen / kAhead) & 1))) break;
          fetch(kbase, kd, seen);
        }
        if (use && !(ok = warp_wait(vfree + 8 * stage, (use - 1) & 1))) break;
        put(v_sm + stage * S::kOperand, vd);
        __syncwarp();
        if (lane == 0) mbar_arrive(vfull + 8 * stage);
        if (more) fetch(vbase, vd, seen);
      }
    }
  } else {
    // ------------------------------------------------ products
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (warp == 18) {
      // ---------------------------------------------- pages and scales of the tiles; lane = block of 16 positions
      const int psh = p.P == 16 ? 4 : p.P == 32 ? 5 : 6;
      unsigned seen = 0;
      bool ok = true;
      for (unsigned seg = 0; ok; ++seg) {
        if (!(ok = warp_wait(segfull + 8 * (seg % kSegRing), (seg / kSegRing) & 1))) break;
        const PreSegment& sg = st.seg[seg % kSegRing];
        if (sg.begin < 0) break;
        const int tile0 = sg.tile0, tile1 = sg.tile1, positions = sg.positions, kvh = sg.kvh;
        const int* trow = p.table + (long long)p.groups[sg.begin] * p.ld_table;
        __syncwarp();
        if (lane == 0) mbar_arrive(segfree + 8 * (seg % kSegRing));
        auto page_of = [&](int tile) {
          const int pos = tile * kPreTile + 16 * lane;
          return lane < 8 && pos < positions ? valid_page(__ldg(trow + (pos >> psh)), p.pages) : -1;
        };
        // a tile's page was asked for two tiles ago, its scales one tile ago
        float ks = 0.f, vs = 0.f;
        auto scales = [&](int page) {
          const long long at = (long long)max(page, 0) * p.hkv + kvh;
          ks = page >= 0 ? __ldg(p.kv.ks + at) : 0.f;
          vs = page >= 0 ? __ldg(p.kv.vs + at) : 0.f;
        };
        int page = page_of(tile0), next = page_of(tile0 + 1);
        scales(page);
        for (int tile = tile0; tile < tile1; ++tile, ++seen) {
          const unsigned entry = seen % kAhead;
          if (seen >= kAhead && !(ok = warp_wait(sidefree + 8 * entry, (seen / kAhead - 1) & 1))) break;
          const int later = page_of(tile + 2);
          const float v = fmaxf(vs, kTinyScale);
          if (lane < 8) {
            st.page[entry][lane] = page;
            Block bl;
            bl.k = ks;
            bl.lv = __log2f(v);
            bl.rv = 1.f / v;
            bl.unused = 0.f;
            st.side[entry][lane] = bl;
          }
          const unsigned mask = __ballot_sync(0xffffffffu, page >= 0);
          const unsigned most = __reduce_max_sync(0xffffffffu, __float_as_uint(v));  // lanes without a block have the least
          if (lane == 0) {
            st.have[entry] = mask;
            st.top[entry] = (int)((most + 0x7fffffu) >> 23) - 127;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(sidefull + 8 * entry);
          page = next;
          scales(page);
          next = later;
        }
      }
    }
    if (warp == 17 && lane == 0) {
      // ---------------------------------------------- segments of this CTA's run
      // A unit is kPreCost, then one cell per tile (two where both slots take every tile: such a tile belongs to the
      // run that has its second cell).
      const unsigned total = st.prefix[ng], per = max((total + gridDim.x - 1) / gridDim.x, (unsigned)kPreMin);
      unsigned at = min((unsigned)min((unsigned long long)per * blockIdx.x, 0xffffffffull), total);
      const unsigned end = min(at + per, total);
      unsigned seg = 0;
      bool ok = true;
      auto place = [&]() -> bool { return seg < kSegRing || wait(segfree + 8 * (seg % kSegRing), (seg / kSegRing - 1) & 1); };
      while (at < end && ok) {
        int lo = 0, hi = ng - 1;  // the last group that starts at or before `at`
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (st.prefix[mid] <= at) lo = mid;
          else hi = mid - 1;
        }
        const int positions = st.positions[lo];
        const unsigned tiles = (unsigned)(positions + kPreTile - 1) / kPreTile;
        const unsigned rows = (unsigned)(p.groups[2 * p.B + lo] * p.T * p.G), pairs = rows / kUnitRows, rest = rows % kUnitRows;
        const unsigned pair_cost = 2 * tiles + kPreCost, rest_cost = rest ? (rest > kSlotRows ? 2 : 1) * tiles + kPreCost : 0;
        const unsigned head_cost = pairs * pair_cost + rest_cost, x = at - st.prefix[lo], head = x / head_cost;
        if (head >= (unsigned)p.hkv) break;  // cannot be
        const unsigned unit = min((x - head * head_cost) / pair_cost, pairs);
        PreSegment sg;
        sg.begin = p.groups[p.B + lo];
        sg.positions = positions;
        sg.kvh = (int)head;
        sg.rows0 = (int)(unit * kUnitRows);
        sg.rows = (int)(unit < pairs ? kUnitRows : rest);
        sg.both = sg.rows > kSlotRows;
        const int w = sg.both ? 2 : 1;
        const unsigned r0 = st.prefix[lo] + head * head_cost + unit * pair_cost + kPreCost, u1 = r0 + w * tiles;
        const unsigned from = max(at, r0), to = min(end, u1);
        at = to > at ? to : end;
        if (from >= to) continue;
        sg.tile0 = (int)((from - r0) / w);
        sg.tile1 = (int)((to - r0) / w);
        if (sg.tile0 >= sg.tile1) continue;
        if (sg.tile0 == 0) {
          const int u = unit_base(p, lo, sg.begin) + sg.kvh * (int)((rows + kUnitRows - 1) / kUnitRows) + (int)unit;
          p.parts.units[u] = make_int4((int)((r0 + w - 1) / per), (int)((u1 - 1) / per), sg.both, 0);
        }
        if (!(ok = place())) break;
        st.seg[seg % kSegRing] = sg;
        mbar_arrive(segfull + 8 * (seg % kSegRing));
        ++seg;
      }
      if (ok && place()) {
        st.seg[seg % kSegRing].begin = -1;
        mbar_arrive(segfull + 8 * (seg % kSegRing));
      }
    }
    if (warp == 16) {
      // The whole warp walks along, so that addresses stay uniform; one lane issues.  A segment's tiles take the stages in
      // turn from the first one on, and each step is compiled for its stage: descriptors are sums of constants.
      const bool leader = elect_one();
      unsigned uses0 = 0, uses1 = 0, p0 = 0, p1 = 0, seen = 0;  // of the stages; weights waited for, by slot; tiles
      bool ok = tmem == 0;                            // all columns were asked for
      auto uses = [&](int stage) -> unsigned& { return stage ? uses1 : uses0; };
      // S of slot s from a stage's K and a slot's Q; S's P of the tile before has been taken up by an earlier product
      auto first_product = [&](auto s, auto stage, auto q) {
        if (leader) {
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) {
            const uint32_t off = (i >> 2) * S::kHalf + (i & 3) * 32;
            mma_ss(S::s_at(s.value), operand(q_sm + q.value * S::kOperand + off, 16), operand(k_sm + stage.value * S::kOperand + off, 16),
                   instruction(kPreTile, false), i > 0);
          }
          tc_commit(sfull + 8 * s.value);
        }
      };
      auto second_product = [&](auto s, auto stage, bool more) -> bool {
        if (!warp_wait(pfull + 8 * s.value, (s.value ? p1++ : p0++) & 1)) return false;
        tc_after();
        if (leader) {
#pragma unroll
          for (int i = 0; i < kPreTile / 16; ++i)
            mma_ts(S::o_at(s.value), S::p_at(s.value) + 8 * i, operand(v_sm + stage.value * S::kOperand + i * 2048, S::kHalf),
                   instruction(HD, true), more || i > 0);
        }
        return true;
      };
      // use u of a stage's K or V
      auto ready = [&](uint32_t bar, unsigned u) -> bool {
        if (!warp_wait(bar, u & 1)) return false;
        tc_after();
        return true;
      };
      auto release = [&](uint32_t bar) {
        if (leader) tc_commit(bar);
      };
      // a tile's weights have been made, and its codes had been loaded before: its pages and scales are done with
      auto forget = [&]() {
        if (leader) mbar_arrive(sidefree + 8 * (seen % kAhead));
        ++seen;
      };
      const std::integral_constant<int, 0> zero;
      const std::integral_constant<int, 1> one;
      // tile i of n, in `stage`; the other stage takes the next one
      auto both_step = [&](auto stage, auto other, unsigned i, unsigned n) -> bool {
        if (!ready(vfull + 8 * stage.value, uses(stage.value) + (i >> 1)) || !second_product(zero, stage, i > 0)) return false;
        if (i + 1 < n) {
          if (!ready(kfull + 8 * other.value, uses(other.value) + ((i + 1) >> 1))) return false;
          first_product(zero, other, zero);
        }
        if (!second_product(one, stage, i > 0)) return false;
        forget();
        release(vfree + 8 * stage.value);
        if (i + 1 < n) {
          first_product(one, other, one);
          release(kfree + 8 * other.value);
        }
        return true;
      };
      // tile i of n, in stage and slot i % 2; the stage's next tile follows
      auto alone_step = [&](auto stage, unsigned i, unsigned n) -> bool {
        if (!ready(vfull + 8 * stage.value, uses(stage.value) + (i >> 1)) || !second_product(stage, stage, i > 1)) return false;
        forget();
        release(vfree + 8 * stage.value);
        if (i + 2 < n) {
          if (!ready(kfull + 8 * stage.value, uses(stage.value) + (i >> 1) + 1)) return false;
          first_product(stage, stage, zero);
          release(kfree + 8 * stage.value);
        }
        return true;
      };
      for (unsigned seg = 0; ok; ++seg) {
        if (!(ok = warp_wait(segfull + 8 * (seg % kSegRing), (seg / kSegRing) & 1))) break;
        const PreSegment& sg = st.seg[seg % kSegRing];
        if (sg.begin < 0) break;
        const unsigned n = (unsigned)(sg.tile1 - sg.tile0);
        const int both = sg.both;
        __syncwarp();
        if (lane == 0) mbar_arrive(segfree + 8 * (seg % kSegRing));
        if (!(ok = warp_wait(qfull, seg & 1) && warp_wait(qfull + 8, seg & 1) && ready(kfull, uses0))) break;
        first_product(zero, zero, zero);
        if (both) {
          first_product(one, zero, one);
          release(kfree);
          for (unsigned i = 0; i < n && ok; i += 2) {
            ok = both_step(zero, one, i, n);
            if (ok && i + 1 < n) ok = both_step(one, zero, i + 1, n);
          }
        } else {
          release(kfree);
          if (n > 1) {
            if (!(ok = ready(kfull + 8, uses1))) break;
            first_product(one, one, zero);
            release(kfree + 8);
          }
          for (unsigned i = 0; i < n && ok; i += 2) {
            ok = alone_step(zero, i, n);
            if (ok && i + 1 < n) ok = alone_step(one, i + 1, n);
          }
        }
        if (!ok) break;
        release(oend);
        uses0 += (n + 1) >> 1;
        uses1 += n >> 1;
      }
      // nothing may be in flight when tensor memory is given back
      if (leader) tc_commit(drained);
      const uint64_t t0 = globaltimer();
      while (!mbar_try(drained, 0) && globaltimer() - t0 < kWaitNs) {
      }
      if (tmem != 0 && p.status) *p.status = 1;
    }
    __syncwarp();
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == 16)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// Parts of the workspace behind the second kernel's.
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

struct SharedLayout {
  size_t later, later_stats, first, first_stats, rows, units, total;
  int max_units;
};

// max_units is 0 where a call is too large for the units' numbers.
SharedLayout shared_layout(const wal_kv8_cache* cache, int64_t B, int64_t T, int32_t hq) {
  const size_t grid = (size_t)sm_count(), rows = (size_t)B * T * hq, hd = (size_t)cache->head_dim;
  const int64_t units = cache->kv_heads * (B / 2 + B * T * (hq / cache->kv_heads) / kUnitRows + 2);
  SharedLayout l;
  l.max_units = units < 0x7fffffff ? (int)units : 0;
  l.later = align256(attention_workspace(cache, B, T, hq));
  l.later_stats = l.later + grid * 2 * kSlotRows * hd * sizeof(float);
  l.first = align256(l.later_stats + grid * 2 * kSlotRows * sizeof(float2));
  l.first_stats = l.first + rows * 2 * hd * sizeof(float);
  l.rows = align256(l.first_stats + rows * 2 * sizeof(float2));
  l.units = l.rows + (size_t)B * sizeof(int4);
  l.total = align256(l.units + (size_t)units * sizeof(int4));
  return l;
}

template <int HD, int KIND>
int launch_prefix(const PreParams& p, cudaStream_t st) {
  auto kern = kv8_prefix_kernel<HD, KIND>;
  static std::atomic<uint64_t> allowed{0};  // devices where the kernel may use its shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return WAL_ERR_CUDA;
  if (!(allowed.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PreShape<HD>::kSmem) != cudaSuccess) return WAL_ERR_CUDA;
    allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  return launch_chain(kern, dim3((unsigned)sm_count()), kPreThreads, PreShape<HD>::kSmem, st, p);
}

}  // namespace

extern "C" {

size_t wal_kv8_attention_shared_workspace(const wal_kv8_cache* cache, int64_t B, int64_t T, int32_t hq) {
  if (attention_workspace(cache, B, T, hq) == 0 || B > kMaxShared || B * T > 0x7fffffff / hq) return 0;
  const SharedLayout l = shared_layout(cache, B, T, hq);
  return l.max_units ? l.total : 0;
}

int wal_kv8_attention_shared(const wal_kv8_cache* cache, int32_t layer, const uint16_t* q, int64_t ld_q, int64_t B, int64_t T,
                             int32_t hq, const int32_t* table, int64_t ld_table, int64_t max_pages, const int32_t* lens,
                             const int32_t* new_lens, const int32_t* groups, float scale, uint16_t* out, int64_t ld_out,
                             void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  Plan plan = {};
  const int st = make_plan(cache, layer, q, ld_q, B, T, hq, table, ld_table, max_pages, lens, new_lens, scale, out, ld_out,
                           workspace, workspace_bytes, &plan);
  if (st != WAL_OK) return st;
  if (!groups) return WAL_ERR_INVALID_ARGUMENT;
  if (B > kMaxShared) return WAL_ERR_SHAPE;
  const SharedLayout l = shared_layout(cache, B, T, hq);
  // the sums of costs fit 32 bits, whatever the lengths
  if (!l.max_units || l.max_units * (2 * (max_pages * plan.p.P / kPreTile + 1) + kPreCost) >= (1LL << 31)) return WAL_ERR_SHAPE;
  if (workspace_bytes < l.total) return WAL_ERR_BUFFER_TOO_SMALL;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const AttnParams& a = plan.p;
  PreParams p = {};
  p.q = q;
  p.ld_q = ld_q;
  p.kv = a.kv;
  p.B = a.B;
  p.T = a.T;
  p.hq = hq;
  p.hkv = a.hkv;
  p.G = a.G;
  p.P = a.P;
  p.pages = a.pages;
  p.max_pages = a.max_pages;
  p.table = table;
  p.ld_table = ld_table;
  p.new_lens = new_lens;
  p.groups = groups;
  p.qscale = a.qscale;
  p.parts.first = reinterpret_cast<float*>(ws + l.first);
  p.parts.first_stats = reinterpret_cast<float2*>(ws + l.first_stats);
  p.parts.later = reinterpret_cast<float*>(ws + l.later);
  p.parts.later_stats = reinterpret_cast<float2*>(ws + l.later_stats);
  p.parts.rows = reinterpret_cast<int4*>(ws + l.rows);
  p.parts.units = reinterpret_cast<int4*>(ws + l.units);
  p.parts.max_units = l.max_units;
  p.parts.ctas = sm_count();
  p.status = status;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  int rc;
  if (cache->head_dim == 128) rc = cache->kind == WAL_KV_INT8 ? launch_prefix<128, WAL_KV_INT8>(p, s) : launch_prefix<128, WAL_KV_E4M3>(p, s);
  else rc = cache->kind == WAL_KV_INT8 ? launch_prefix<64, WAL_KV_INT8>(p, s) : launch_prefix<64, WAL_KV_E4M3>(p, s);
  if (rc != WAL_OK) return rc;
  plan.p.from = groups + 3 * B;
  plan.p.parts = p.parts;
  return launch_plan<true>(plan, cache->head_dim, cache->kind, s);
}

}  // extern "C"
