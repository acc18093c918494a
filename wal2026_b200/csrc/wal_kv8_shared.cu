// Attention over the paged 8-bit KV cache for rows that share their first
// positions: what a group shares is read once for all of its rows.
//
// Two kernels.  The first one attends all query rows of a group (members x T tokens
// x G heads of a kv head, 128 to a tile) to the shared positions and leaves, for
// every row and head, (reference exponent, sum, weighted sum) in the workspace; the
// second one is the attention of wal_kv8_attn.cuh over each row's own positions,
// which adds the two.  Shared positions lie before every row's own, so
// there is no causal mask.
//
// The first kernel: a group of many samples has hundreds of rows per kv head, so
// its products run on the tensor cores by tcgen05 with both codes and weights as
// f16 (an int8 or e4m3 code is exact in f16).  Per 128 positions, S = Q K^T
// (128 x 128 x HD) and O += P V; Q is scaled by a power of two per row into f16's range, K codes
// and V codes stand in shared memory as f16 rows of positions (K-major for the
// first product, MN-major for the second: the same layout), S and O live in tensor
// memory, and P is written there too, as the A operand of the second product.
//   warps 0-3   a query row per thread: maximum, exponentials, sums, P, and the
//               rescaling of O where the running maximum has grown by 2^8
//   warps 4-11  codes from global memory through registers (loads run ahead of the
//               tile being converted) to f16 in shared memory, two stages
//   warp 12     issues the products
// P is exp2(x - m + 7) times the block's V scale over the largest V scale so far:
// at most 2^15, so that f16 keeps weights down to 2^-32 of the largest; each is
// rounded by 2^-12 at most.  Maxima, sums and outputs are fp32.
//
// The position tiles of all (row tile, kv head) units are cut into equal runs, one
// per SM; runs that share a unit leave partial results, and the last of them to
// finish joins them in order.  Every wait is bounded by a deadline.
#include "wal_kv8_attn.cuh"

#include <type_traits>

namespace {

constexpr int kSoftWarps = 4, kLoadWarps = 8;
constexpr int kPreThreads = 32 * (kSoftWarps + kLoadWarps + 1);
constexpr int kPreTile = 128;       // positions
constexpr int kPreRows = 128;       // query rows
constexpr int kPreCost = 4;         // what starting and ending a unit costs, in tiles
constexpr int kPreMin = 1;          // least tiles of a run
constexpr int kMaxGroups = 2048;
constexpr int kMaxShared = 4096;    // rows of a call
constexpr unsigned long long kWaitNs = 2000000000ull;  // 2 s per wait, then give up
constexpr float kShift = 7.f;       // weights are 2^7 times exp2(x - m)

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
  float* pre;         // [B * T][hq][HD]
  float2* pre_stats;  // [B * T][hq]
  unsigned* counter;  // [grid]
  float* part;        // [grid][2][128][HD]
  float2* stats;      // [grid][2][128]
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
// One statement for the load and its wait, so that no use of the registers comes between the two.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
        "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
        "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};\n" ::"r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
      "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
      "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]),
      "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n" ::"r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
      "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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
  static constexpr int kHalf = kPreTile * 128;            // 64 columns of 128 rows
  static constexpr int kOperand = kHalf * (HD / 64);      // Q, a stage of K, a stage of V
  static constexpr int kStages = 2;
  static constexpr int kSmem = 1024 + kOperand * (1 + 2 * kStages);
  static constexpr int kS = 0, kPm = 256, kO = 384;       // tensor memory columns: S twice, P twice, O
};

// A unit's tiles that one CTA takes.
struct PreSegment {
  int begin, size;    // members in groups[0]
  int positions;      // shared
  int rt, kvh;
  int tile0, tile1;
  bool whole, leads;
  long long r0, u1;   // the unit's first tile and end on the line of all tiles
};

struct PreState {
  long long prefix[kMaxGroups + 1];  // cost before each group
  float side[4][2][8];               // K and V scales of a tile's blocks of 16 positions
  unsigned have[4];                  // blocks that have a page
  long long wsum[kPreThreads / 32];
  unsigned long long bars[24];
  uint32_t tmem;
  int abort;
  int last;
};

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

template <int HD, int KIND>
__global__ void __launch_bounds__(kPreThreads, 1) kv8_prefix_kernel(const __grid_constant__ PreParams p) {
  using S = PreShape<HD>;
  constexpr int PIECES = HD / 16, PER = kPreTile * PIECES / (32 * kLoadWarps);  // 16-byte pieces of a row; per thread
  extern __shared__ uint8_t smem_raw[];
  __shared__ PreState st;
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  const uint32_t q_sm = base, k_sm = q_sm + S::kOperand, v_sm = k_sm + S::kStages * S::kOperand;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t bars = smem_u32(st.bars);
  const uint32_t kfull = bars, vfull = bars + 16, kfree = bars + 32, vfree = bars + 48, sfull = bars + 64, pfull = bars + 80;
  const uint32_t odone = bars + 96, qfull = bars + 112, drained = bars + 120, joined = bars + 128, sidefull = bars + 136;
  volatile int* const abort = &st.abort;

  if (tid == 0) {
    st.abort = 0;
    for (int s = 0; s < 2; ++s) {
      mbar_init(kfull + 8 * s, kLoadWarps);
      mbar_init(vfull + 8 * s, kLoadWarps);
      mbar_init(kfree + 8 * s, 1);
      mbar_init(vfree + 8 * s, 1);
      mbar_init(sfull + 8 * s, 1);
      mbar_init(pfull + 8 * s, kSoftWarps);
      mbar_init(odone + 8 * s, 1);
    }
    mbar_init(qfull, kSoftWarps);
    mbar_init(drained, 1);
    mbar_init(joined, kSoftWarps);
    for (int s = 0; s < 4; ++s) mbar_init(sidefull + 8 * s, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&st.tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  chain();
  // cost of the groups and their running sum
  {
    const int ng = min(p.B / 2, kMaxGroups), each = (ng + kPreThreads - 1) / kPreThreads, i0 = min(tid * each, ng), i1 = min(i0 + each, ng);
    auto cost = [&](int i) -> long long {
      int begin, size, positions;
      if (!group_of(p, i, begin, size, positions)) return 0;
      const long long rt = ((long long)size * p.T * p.G + kPreRows - 1) / kPreRows;
      return rt * p.hkv * ((positions + kPreTile - 1) / kPreTile + kPreCost);
    };
    long long mine = 0;
    for (int i = i0; i < i1; ++i) mine += cost(i);
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
      st.prefix[i] = sum;
      sum += cost(i);
    }
    if (tid == kPreThreads - 1) st.prefix[ng] = sum;
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = st.tmem;
  const int ng = min(p.B / 2, kMaxGroups);
  const long long total = st.prefix[ng];
  const long long per = max((total + gridDim.x - 1) / gridDim.x, (long long)(kPreMin + kPreCost));
  long long at = min(per * blockIdx.x, total);
  const long long run0 = at, end = min(at + per, total);

  // the next segment of this CTA's run; every role walks the same list
  auto next = [&](PreSegment& sg) -> bool {
    while (at < end) {
      int lo = 0, hi = ng - 1;  // the last group that starts at or before `at`
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (st.prefix[mid] <= at) lo = mid;
        else hi = mid - 1;
      }
      if (!group_of(p, lo, sg.begin, sg.size, sg.positions)) return false;  // cannot be: it has a cost
      const int tiles = (sg.positions + kPreTile - 1) / kPreTile;
      const long long rts = ((long long)sg.size * p.T * p.G + kPreRows - 1) / kPreRows;
      const long long unit = (at - st.prefix[lo]) / (tiles + kPreCost);
      sg.kvh = (int)(unit / rts);
      sg.rt = (int)(unit % rts);
      sg.r0 = st.prefix[lo] + unit * (tiles + kPreCost) + kPreCost;
      sg.u1 = sg.r0 + tiles;
      const long long from = max(at, sg.r0), to = min(end, sg.u1);
      sg.leads = from == run0;
      at = min(end, sg.u1);
      if (from >= to) continue;
      sg.tile0 = (int)(from - sg.r0);
      sg.tile1 = (int)(to - sg.r0);
      sg.whole = from == sg.r0 && to == sg.u1;
      return true;
    }
    return false;
  };
  auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
    if (mbar_try(bar, parity)) return true;
    const uint64_t t0 = globaltimer();
    while (!mbar_try(bar, parity)) {
      if (*abort) return false;
      if (globaltimer() - t0 > kWaitNs) {
        *abort = 1;
        if (p.status) *p.status = 1;
        return false;
      }
    }
    return true;
  };

  // the same for all lanes of a warp
  auto warp_wait = [&](uint32_t bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, wait(bar, parity)); };

  PreSegment sg;
  unsigned it = 0;  // tiles so far
  if (warp < kSoftWarps) {
    // ------------------------------------------------ softmax: thread = query row
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    unsigned syncs = 0;
    bool ok = true;
    auto soft_sync = [&]() -> bool {  // of the four warps
      __syncwarp();
      if (lane == 0) mbar_arrive(joined);
      return warp_wait(joined, syncs++ & 1);
    };
    while (ok && next(sg)) {
      const long long row = (long long)sg.rt * kPreRows + tid, rows = (long long)sg.size * p.T * p.G;
      const int member = (int)min(row / (p.T * p.G), (long long)sg.size - 1), t = (int)(row / p.G % p.T), g = (int)(row % p.G);
      const int b = p.groups[sg.begin + member];
      const bool real = row < rows && (unsigned)b < (unsigned)p.B && (!p.new_lens || t < p.new_lens[b]);
      const long long m_row = (long long)(real ? b : 0) * p.T + (real ? t : 0);
      const int head = sg.kvh * p.G + g;
      // q, scaled into f16's range
      float unscale = 0.f;
      {
        uint4 w[HD / 8];
        const uint16_t* src = p.q + m_row * p.ld_q + (long long)head * HD;
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
          w[i] = real ? __ldg(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0u, 0u, 0u, 0u);
          const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fmaxf(fabsf(bf16_lo(u[e])), fabsf(bf16_hi(u[e]))));
        }
        const int e2 = min(max(14 + 127 - (int)(__float_as_uint(mx) >> 23), -112), 126);
        const float up = __uint_as_float((uint32_t)(e2 + 127) << 23);
        unscale = p.qscale * __uint_as_float((uint32_t)(127 - e2) << 23);
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
          const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
          uint32_t h[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) h[e] = pack_f16(bf16_lo(u[e]) * up, bf16_hi(u[e]) * up);
          const uint32_t dst = q_sm + (i >> 3) * S::kHalf + tid * 128 + (((i & 7) ^ (tid & 7)) << 4);
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(qfull);
      const bool some = __any_sync(0xffffffffu, real);  // a warp without rows only keeps step
      float m = -INFINITY, l = 0.f, vref = 1e-30f;
      for (int tile = sg.tile0; tile < sg.tile1; ++tile, ++it) {
        const int buf = it & 1;
        if (!(ok = warp_wait(sfull + 8 * buf, (it >> 1) & 1))) break;
        // The second product of tile i - 2 has read P; seen for every tile, so that no phase is mistaken for the one before.
        if (it >= 2 && !(ok = warp_wait(odone + 8 * buf, ((it >> 1) - 1) & 1))) break;
        if (!(ok = warp_wait(sidefull + 8 * (it & 3), (it >> 2) & 1))) break;
        tc_after();
        if (some) {
          const float* ks = st.side[it & 3][0];
          const float* vs = st.side[it & 3][1];
          const unsigned have = st.have[it & 3];
          const uint32_t s_at = lanes + S::kS + 128 * buf;
          const int left = sg.positions - tile * kPreTile;  // a multiple of 32
          float mn = -INFINITY, vmax = 0.f;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (32 * c >= left) break;
            uint32_t x[32];
            tmem_ld32(s_at + 32 * c, x);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (!((have >> (2 * c + h)) & 1)) continue;
              float top = __uint_as_float(x[16 * h]);
#pragma unroll
              for (int e = 1; e < 16; ++e) top = fmaxf(top, __uint_as_float(x[16 * h + e]));
              mn = fmaxf(mn, top * (unscale * ks[2 * c + h]));
              vmax = fmaxf(vmax, vs[2 * c + h]);
            }
          }
          const bool first = tile == sg.tile0;
          if (__any_sync(0xffffffffu, first || mn > m + kSlack || vmax > vref)) {
            const float top = fmaxf(m, mn), vr = vmax > vref ? vref / vmax : 1.f;
            const float al = top == -INFINITY ? 0.f : ex2(m - top);
            vref = fmaxf(vref, vmax);
            m = top;
            l *= al;
            if (!first) {
              // O may be touched once the product before has finished; the next one waits for this tile's P
              if (!(ok = warp_wait(odone + 8 * (buf ^ 1), ((it - 1) >> 1) & 1))) break;
              tc_after();
              const float f = al * vr;
#pragma unroll
              for (int c = 0; c < HD / 32; ++c) {
                uint32_t x[32];
                tmem_ld32(lanes + S::kO + 32 * c, x);
#pragma unroll
                for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
                tmem_st32(lanes + S::kO + 32 * c, x);
              }
            }
          }
          const float off = m == -INFINITY ? 0.f : kShift - m, vinv = 1.f / vref;
          // S * f + off in one rounding, whose reference is -off itself; where m is so large that its own rounding
          // shows in the exponent, the product is rounded as the maximum's was
          auto weights = [&](auto large) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t x[32], w[16];
              if (32 * c < left) tmem_ld32(s_at + 32 * c, x);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const bool in = 32 * c < left && ((have >> (2 * c + h)) & 1);
                const float f = unscale * ks[2 * c + h], vf = vs[2 * c + h] * vinv;
                auto weight = [&](uint32_t score) {
                  const float y = __uint_as_float(score);
                  return in ? ex2(large.value ? __fadd_rn(__fmul_rn(y, f), off) : fmaf(y, f, off)) : 0.f;
                };
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                  const float a = weight(x[16 * h + e]), d = weight(x[16 * h + e + 1]);
                  l += a + d;
                  w[8 * h + e / 2] = pack_f16(a * vf, d * vf);
                }
              }
              tmem_st16(lanes + S::kPm + 64 * buf + 16 * c, w);
            }
          };
          if (__any_sync(0xffffffffu, fabsf(off) > 65536.f)) weights(std::true_type{});
          else weights(std::false_type{});
          tmem_st_wait();
        }
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(pfull + 8 * buf);
      }
      if (!ok) break;
      // the unit's sums: O after its last product
      if (!(ok = warp_wait(odone + 8 * ((it - 1) & 1), ((it - 1) >> 1) & 1))) break;
      tc_after();
      const int slot = 2 * blockIdx.x + (sg.leads ? 0 : 1);
      if (some) {
        float* dst = sg.whole ? p.pre + (m_row * p.hq + head) * HD : p.part + ((long long)slot * kPreRows + tid) * HD;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t x[32];
          tmem_ld32(lanes + S::kO + 32 * c, x);
          if (real)
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              __stcg(reinterpret_cast<float4*>(dst + 32 * c + e),
                     make_float4(__uint_as_float(x[e]) * vref, __uint_as_float(x[e + 1]) * vref, __uint_as_float(x[e + 2]) * vref,
                                 __uint_as_float(x[e + 3]) * vref));
        }
        if (real) {
          const float2 v = make_float2(m == -INFINITY ? 0.f : -(kShift - m), l);
          if (sg.whole) p.pre_stats[m_row * p.hq + head] = v;
          else p.stats[(long long)slot * kPreRows + tid] = v;
        }
      }
      tc_before();
      if (!sg.whole) {
        // the last run of the unit to get here joins them all, in order
        const int c0 = (int)(sg.r0 / per), c1 = (int)((sg.u1 - 1) / per);
        if (!(ok = soft_sync())) break;
        if (tid == 0) {
          unsigned before;
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(p.counter + c0) : "memory");
          st.last = before == (unsigned)(c1 - c0);
          if (st.last) p.counter[c0] = 0u;  // ready for the next call
        }
        if (!(ok = soft_sync())) break;
        if (st.last) {
          const int rows_here = (int)min((long long)kPreRows, rows - (long long)sg.rt * kPreRows);
          for (int i = tid; i < rows_here * (HD / 4); i += 128) {
            const int rr = i / (HD / 4), c = i % (HD / 4);
            const long long r = (long long)sg.rt * kPreRows + rr;
            const int bb = p.groups[sg.begin + (int)(r / (p.T * p.G))], tt = (int)(r / p.G % p.T), gg = (int)(r % p.G);
            if ((unsigned)bb >= (unsigned)p.B || (p.new_lens && tt >= p.new_lens[bb])) continue;
            float M = -INFINITY, L = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int k = c0; k <= c1; ++k) {
              const long long s_at = (long long)(2 * k + (k == c0 && sg.r0 != k * per ? 1 : 0)) * kPreRows + rr;
              const float2 v = __ldcg(p.stats + s_at);
              if (v.y == 0.f) continue;
              const float4 o = __ldcg(reinterpret_cast<const float4*>(p.part) + s_at * (HD / 4) + c);
              const float top = fmaxf(M, v.x), a = ex2(M - top), f = ex2(v.x - top);
              M = top;
              L = fmaf(L, a, f * v.y);
              acc.x = fmaf(acc.x, a, f * o.x);
              acc.y = fmaf(acc.y, a, f * o.y);
              acc.z = fmaf(acc.z, a, f * o.z);
              acc.w = fmaf(acc.w, a, f * o.w);
            }
            const long long dst = ((long long)bb * p.T + tt) * p.hq + sg.kvh * p.G + gg;
            reinterpret_cast<float4*>(p.pre)[dst * (HD / 4) + c] = acc;
            if (c == 0) p.pre_stats[dst] = make_float2(L == 0.f ? 0.f : M, L);
          }
        }
        if (!(ok = soft_sync())) break;  // `last` may be written again
      }
    }
  } else if (warp < kSoftWarps + kLoadWarps) {
    // ------------------------------------------------ codes to f16
    const int ct = tid - 32 * kSoftWarps, piece = ct % PIECES, row0 = ct / PIECES;
    constexpr int STEP = 32 * kLoadWarps / PIECES;  // rows between a thread's pieces
    const int psh = p.P == 16 ? 4 : p.P == 32 ? 5 : 6;
    const long long page_codes = (long long)p.hkv * p.P * HD;
    bool ok = true;
    while (ok && next(sg)) {
      const int* trow = p.table + (long long)p.groups[sg.begin] * p.ld_table;
      const uint8_t* kbase = p.kv.k + (long long)sg.kvh * p.P * HD + piece * 16;
      const uint8_t* vbase = p.kv.v + (long long)sg.kvh * p.P * HD + piece * 16;
      uint4 kd[PER], vd[PER];
      float sk = 0.f, sv = 0.f;  // scales of block `ct` of the tile (threads 0 to 7)
      bool has = false;
      auto page_at = [&](int pos) { return pos < sg.positions ? valid_page(__ldg(trow + (pos >> psh)), p.pages) : -1; };
      auto fetch = [&](int tile) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int pos = tile * kPreTile + row0 + i * STEP, page = page_at(pos);
          const long long off = max(page, 0) * page_codes + (pos & (p.P - 1)) * HD;
          kd[i] = page >= 0 ? __ldg(reinterpret_cast<const uint4*>(kbase + off)) : make_uint4(0u, 0u, 0u, 0u);
          vd[i] = page >= 0 ? __ldg(reinterpret_cast<const uint4*>(vbase + off)) : make_uint4(0u, 0u, 0u, 0u);
        }
        if (ct < 8) {
          const int page = page_at(tile * kPreTile + 16 * ct);
          has = page >= 0;
          const long long at_s = (long long)max(page, 0) * p.hkv + sg.kvh;
          sk = has ? __ldg(p.kv.ks + at_s) : 0.f;
          sv = has ? __ldg(p.kv.vs + at_s) : 0.f;
        }
      };
      auto put = [&](uint32_t stage_sm, const uint4 (&d)[PER]) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int r = row0 + i * STEP;
          uint32_t h[8];
          codes_f16<KIND>(d[i].x, h[0], h[1]);
          codes_f16<KIND>(d[i].y, h[2], h[3]);
          codes_f16<KIND>(d[i].z, h[4], h[5]);
          codes_f16<KIND>(d[i].w, h[6], h[7]);
          const uint32_t dst = stage_sm + (piece >> 2) * S::kHalf + r * 128;
          const int c = 2 * (piece & 3);
          // the upper half's lanes start with the odd piece: no two lanes of eight meet in a bank
          const int odd = HD == 128 ? piece >> 2 : 0;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int which = e ^ odd;
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + (((c + which) ^ (r & 7)) << 4)), "r"(which ? h[4] : h[0]),
                         "r"(which ? h[5] : h[1]), "r"(which ? h[6] : h[2]), "r"(which ? h[7] : h[3])
                         : "memory");
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      };
      fetch(sg.tile0);
      for (int tile = sg.tile0; tile < sg.tile1; ++tile, ++it) {
        const int stage = it & 1;
        if (it >= 2 && !(ok = warp_wait(kfree + 8 * stage, ((it >> 1) - 1) & 1))) break;
        put(k_sm + stage * S::kOperand, kd);
        // Scales of a tile stay for four: the tile that takes their place is converted after the second
        // product before it has been issued, and so after its softmax.
        if (ct < 8) {
          st.side[it & 3][0][ct] = sk;
          st.side[it & 3][1][ct] = sv;
          const unsigned mask = __ballot_sync(0xffu, has);
          if (ct == 0) st.have[it & 3] = mask;
        }
        __syncwarp();
        if (ct == 0) mbar_arrive(sidefull + 8 * (it & 3));
        if (lane == 0) mbar_arrive(kfull + 8 * stage);
        if (it >= 2 && !(ok = warp_wait(vfree + 8 * stage, ((it >> 1) - 1) & 1))) break;
        put(v_sm + stage * S::kOperand, vd);
        __syncwarp();
        if (lane == 0) mbar_arrive(vfull + 8 * stage);
        if (tile + 1 < sg.tile1) fetch(tile + 1);
      }
    }
  } else {
    // ------------------------------------------------ products
    if (lane == 0) {
      unsigned seg = 0;
      bool ok = true;
      // S of tile i (stage and buffer i % 2)
      auto first_product = [&](unsigned i) -> bool {
        const unsigned s = i & 1;
        if (!wait(kfull + 8 * s, (i >> 1) & 1)) return false;
        if (i >= 2 && !wait(pfull + 8 * s, ((i >> 1) - 1) & 1)) return false;  // S and P of tile i - 2 have been read and written
        tc_after();
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          mma_ss(tmem + S::kS + 128 * s, operand(q_sm + (k >> 2) * S::kHalf + (k & 3) * 32, 16),
                 operand(k_sm + s * S::kOperand + (k >> 2) * S::kHalf + (k & 3) * 32, 16), instruction(kPreTile, false), k > 0);
        tc_commit(kfree + 8 * s);
        tc_commit(sfull + 8 * s);
        return true;
      };
      while (ok && next(sg)) {
        if (!(ok = wait(qfull, seg & 1))) break;
        ++seg;
        if (!(ok = first_product(it))) break;
        for (int tile = sg.tile0; tile < sg.tile1; ++tile, ++it) {
          if (tile + 1 < sg.tile1 && !(ok = first_product(it + 1))) break;
          const unsigned s = it & 1;
          if (!(ok = wait(vfull + 8 * s, (it >> 1) & 1))) break;
          if (!(ok = wait(pfull + 8 * s, (it >> 1) & 1))) break;
          tc_after();
#pragma unroll
          for (int k = 0; k < kPreTile / 16; ++k)
            mma_ts(tmem + S::kO, tmem + S::kPm + 64 * s + 8 * k, operand(v_sm + s * S::kOperand + k * 2048, S::kHalf), instruction(HD, true),
                   tile > sg.tile0 || k > 0);
          tc_commit(vfree + 8 * s);
          tc_commit(odone + 8 * s);
        }
      }
      // nothing may be in flight when tensor memory is given back
      tc_commit(drained);
      const uint64_t t0 = globaltimer();
      while (!mbar_try(drained, 0) && globaltimer() - t0 < kWaitNs) {
      }
    }
    __syncwarp();
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (warp == 12)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// Parts of the workspace behind the second kernel's.
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

struct SharedLayout {
  size_t counter, part, stats, pre, pre_stats, total;
};

SharedLayout shared_layout(const wal_kv8_cache* cache, int64_t B, int64_t T, int32_t hq) {
  const size_t grid = (size_t)sm_count(), rows = (size_t)B * T * hq, hd = (size_t)cache->head_dim;
  SharedLayout l;
  l.counter = align256(attention_workspace(cache, B, T, hq));
  l.part = l.counter + align256(grid * sizeof(unsigned));
  l.stats = l.part + grid * 2 * kPreRows * hd * sizeof(float);
  l.pre = align256(l.stats + grid * 2 * kPreRows * sizeof(float2));
  l.pre_stats = l.pre + rows * hd * sizeof(float);
  l.total = align256(l.pre_stats + rows * sizeof(float2));
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
  return shared_layout(cache, B, T, hq).total;
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
  p.pre = reinterpret_cast<float*>(ws + l.pre);
  p.pre_stats = reinterpret_cast<float2*>(ws + l.pre_stats);
  p.counter = reinterpret_cast<unsigned*>(ws + l.counter);
  p.part = reinterpret_cast<float*>(ws + l.part);
  p.stats = reinterpret_cast<float2*>(ws + l.stats);
  p.status = status;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  int rc;
  if (cache->head_dim == 128) rc = cache->kind == WAL_KV_INT8 ? launch_prefix<128, WAL_KV_INT8>(p, s) : launch_prefix<128, WAL_KV_E4M3>(p, s);
  else rc = cache->kind == WAL_KV_INT8 ? launch_prefix<64, WAL_KV_INT8>(p, s) : launch_prefix<64, WAL_KV_E4M3>(p, s);
  if (rc != WAL_OK) return rc;
  plan.p.from = groups + 3 * B;
  plan.p.pre = p.pre;
  plan.p.pre_stats = p.pre_stats;
  return launch_plan<true>(plan, cache->head_dim, cache->kind, s);
}

}  // extern "C"
