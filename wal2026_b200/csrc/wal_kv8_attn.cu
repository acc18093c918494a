// Attention of new tokens over the paged 8-bit KV cache (grouped-query heads).
//
//   out[b, t, h] = sum_j softmax_j(scale * q[b, t, h] . k_j) v_j,  j <= lens[b] + t
//
// The cache is read once per kv head and row tile; everything else is small, so
// the kernel is built to keep loads in flight and bytes per value at one.
//
// Work split.  The rows that share a kv head (T tokens x G heads, row t * G + g)
// form tiles of 8 to 96 rows; a unit is one (sequence, row tile, kv head)
// over its positions in tiles of 32.  The position tiles of all units, in
// order, are cut into equal runs, one per CTA of a grid that fills the GPU
// once, whatever the mix of lengths: every CTA reads the lengths, sums the tile
// counts and finds its run.  A unit that one CTA covers is written by it; one
// that several cover leaves (max, sum, un-normalised output) per row in the
// workspace, and the last of its CTAs to arrive joins them in CTA order, so
// results do not depend on timing.  Starting and ending a unit costs a CTA about
// as much as eight tiles, which the runs count (48 sequences of 0 to 4096
// positions: 67 us without, 48.6 us with), and a short unit is not split (64
// sequences of 256: 19.7 us split, 17.9 us whole; one sequence of 512 loses, 8.3
// us split and 10.0 us whole).  Calls of more than kMaxEntries
// (sequence, row tile) pairs have units enough to give each CTA whole ones.
//
// Within a CTA.  One warp group (one warp for each 8, 16 or 24 rows) takes every NS-th
// position tile through its own ring of stages in shared memory (16-byte
// asynchronous copies, page by page; pieces swizzled so that the matrix loads
// below meet no bank conflict), with its own running maximum and sum.  Codes
// become 16-bit floats in registers (each int8 and e4m3 code is exact in f16
// and in bf16) and feed mma.sync m16n8k16 with fp32 accumulators.  K fragments
// come from ldmatrix (four dims of a token per register), V fragments from the
// transposing 8-bit ldmatrix (four tokens of a dim per register); the order of
// k within a fragment is free, so Q and P are laid out to match.
//
// Numerics.  q is scaled by a power of two per row into f16's range: elements
// down to 2^-31 of the row's largest keep all of bf16's bits.  Scores, maxima,
// sums and outputs are fp32.  P, times the block's V scale over the largest V
// scale seen so far (which moves with the running maximum), enters the second
// product as the sum of two bf16 numbers: 2^-16 of each weight at most and fp32's
// range, where one f16 would lose weights below 2^-24 of the largest and one
// bf16 would add an error the size of the output's own rounding.
// Scores and weights are computed transposed (tokens or dims are the 16 rows of a
// tensor-core tile, query rows its 8 columns), so that eight rows waste nothing.
//
// Bounds, on B200 (1965 MHz unless said).  4 sequences of 100001 to 131071
// positions (983 MB), 64 query and 8 kv heads of 128, int8: 157 us in a burst,
// 6.2 TB/s of cache, 95% of a copy's rate (4 x 131072: 171 us, the same rate);
// under a second of it the power limit lowers the clock to 1.6 GHz and the
// conversions of the codes (five instructions for four K codes, seven for four V
// codes, 830 instructions per warp and tile in all) make it 189 us.  Small calls
// are a chain of latencies: lengths 2 us, pages and first tile 2.5 us, joining
// runs 3 us; one sequence of 2048 takes 10.0 us where its bytes take 0.6.  More
// rows add products: 16 sequences of 4300 on average with 8 / 16 / 24 / 32 / 64
// rows per kv head take 36 / 48 / 61 / 82 / 149 us (memory: 22), bound by the
// instructions of conversions and products, which dependent chains at two warps per
// scheduler issue at half rate.
// Measured slower, with earlier forms of the kernel (61 us for 24 rows, 82 for 32,
// 162 for the long sequences): the two products of a tile split between two warps
// that pass weights through shared memory (24 rows 69 us); four warps of eight
// rows, each converting for itself (32 rows 108 us); 3 stages and 2 CTAs per SM
// for 8 rows (168 us against 162); three 8-bit digits of q times K codes in
// integers, which needs no conversion of K (187 us sustained against 190, but
// 11.1 us for the single sequence).
#include "wal_kv8.cuh"

#include <cuda_fp16.h>

namespace {

using namespace wal_kv8;

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 32;          // positions of a tile
constexpr int kMaxEntries = 1024;  // (sequence, row tile) pairs of a balanced call
constexpr int kMinTiles = 4;       // least tiles of a run: one per warp (one sequence of 2048: 10.0 us, 10.8 with 8; of 8192: 15.3 and 13.7)
constexpr int kUnitCost = 8;       // what starting and ending a unit costs, in tiles
constexpr unsigned kWholeCost = 28;  // units of at most this cost are not split
constexpr float kSlack = 8.f;      // weights may reach 2^8 before the running maximum moves

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&m)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3])
               : "r"(addr));
}
// Two 16 x 16 byte matrices, transposed: register 2i holds column lane / 4 of
// matrix i, rows 4 * (lane % 4) .. + 3; register 2i + 1 column 8 + lane / 4.
__device__ __forceinline__ void ldsm_t8_x2(uint32_t addr, uint32_t (&m)[4]) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3])
               : "r"(addr));
}

// The transpose of an 8 x 8 matrix of 16-bit values, two neighbours of a row per lane.
__device__ __forceinline__ uint32_t transpose(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t v;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  return v;
}

// Which of a register's four codes share a 16-bit pair: bytes (0, 2) and (1, 3),
// as masks split even from odd bytes, but (0, 1) and (2, 3) where e4m3 becomes
// f16 by the conversion that takes neighbours.
__host__ __device__ constexpr int split_at(int pair, int e) { return 2 * e + pair; }
template <int KIND>
__host__ __device__ constexpr int k_at(int pair, int e) {
  return KIND == WAL_KV_INT8 ? split_at(pair, e) : 2 * pair + e;
}

// Bit patterns of the conversions, passed as a parameter: a three-input logic
// instruction takes one immediate, and two known constants cost a move each time.
struct Masks {
  uint32_t low8 = 0x00ff00ffu, f16_128 = 0x64806480u;                       // 1024 + code + 128 as f16
  uint32_t low7 = 0x007f007fu, bit7 = 0x00800080u, bf16_128 = 0x43004300u;  // 128 as bf16
};

template <int LUT>
__device__ __forceinline__ uint32_t lop3(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, %4;" : "=r"(r) : "r"(a), "r"(b), "r"(c), "n"(LUT));
  return r;
}
constexpr int kAndOr = 0xea, kAndXor = 0x6a;  // (a & b) | c, (a & b) ^ c

// K codes as f16.
template <int KIND>
__device__ __forceinline__ void to_f16(const Masks& k, uint32_t w, uint32_t& p0, uint32_t& p1) {
  if (KIND == WAL_KV_INT8) {
    // 0x6400 | u is 1024 + u; u = code + 128
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(p0) : "r"(lop3<kAndXor>(w, k.low8, k.f16_128)), "r"(k.f16_128));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(p1) : "r"(lop3<kAndXor>(w >> 8, k.low8, k.f16_128)), "r"(k.f16_128));
  } else {
    asm("{.reg .b16 lo, hi;\n mov.b32 {lo, hi}, %2;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n cvt.rn.f16x2.e4m3x2 %1, hi;\n}"
        : "=r"(p0), "=r"(p1)
        : "r"(w));
  }
}

// V codes as bf16: int8 as they are, e4m3 times 2^-120.  Weights take v_unit of
// that back, which leaves them room for 2^kSlack and a rounding (the largest bf16
// number is just below 2^128), and the finished outputs take v_rest.
template <int KIND>
__host__ __device__ constexpr float v_unit() {
  return KIND == WAL_KV_INT8 ? 1.f : 5.192296858534828e33f;  // 2^112
}
template <int KIND>
__host__ __device__ constexpr float v_rest() {
  return KIND == WAL_KV_INT8 ? 1.f : 256.f;
}
static_assert(kSlack <= 8.f, "a weight of 2^kSlack * 2^112 stays far from the largest bf16 number");
template <int KIND>
__device__ __forceinline__ void to_bf16(const Masks& k, uint32_t w, uint32_t& p0, uint32_t& p1) {
  if (KIND == WAL_KV_INT8) {
    // 0x4300 | low seven bits is 128 + them; 0x4300 | sign bit is 128 or 256
    const uint32_t v = w >> 8;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(p0) : "r"(lop3<kAndOr>(w, k.low7, k.bf16_128)), "r"(lop3<kAndOr>(w, k.bit7, k.bf16_128)));
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(p1) : "r"(lop3<kAndOr>(v, k.low7, k.bf16_128)), "r"(lop3<kAndOr>(v, k.bit7, k.bf16_128)));
  } else {
    // exponent and fraction bits moved to bf16's: the value times 2^(7 - 127),
    // subnormals included, and finite for every byte
    p0 = ((w << 8) & 0x80008000u) | ((w << 4) & 0x07f007f0u);
    p1 = (w & 0x80008000u) | ((w >> 4) & 0x07f007f0u);
  }
}

struct AttnParams {
  const uint16_t* q;
  long long ld_q;
  LayerView kv;
  int B, T, hq, hkv, G, P, pages, max_pages;
  int row_tiles;  // per (sequence, kv head)
  const int* table;
  long long ld_table;
  const int* lens;
  const int* new_lens;
  float qscale;  // scale * log2(e)
  uint16_t* out;
  long long ld_out;
  unsigned* counter;  // [grid] of the unit that starts in a CTA's run and goes on past it
  float* part;        // [grid][2][rows][HD]
  float2* stats;      // [grid][2][rows] (max, sum)
  unsigned units;  // (sequence, row tile, kv head)
  bool balanced;
  Masks masks;
};

// A tile's rows stand HD bytes apart; their 16-byte pieces are permuted within
// 128-byte lines by xor with a key of the row, distinct among the eight rows
// that one matrix load reads together (K: rows 4 * (i / 2) + 2 * (i % 2) + s,
// V: eight in a row).  Keys are linear in the bits of the row, so that offsets
// of a lane's rows differ by an xor and an addition of constants.
__device__ __forceinline__ constexpr uint32_t k_key(int r) { return (uint32_t)((r >> 1) & 7) << 4; }
template <int HD>
__device__ __forceinline__ constexpr uint32_t v_key(int r) {
  return (uint32_t)(HD == 128 ? r & 7 : (r >> 1) & 3) << 4;
}

// RW rows per warp (8, 16 or 24), WM warps per group.
template <int HD, int RW, int WM>
struct Shape {
  static constexpr int kRows = RW * WM;         // query rows of a unit
  static constexpr int NS = kWarps / WM;        // warp groups
  static constexpr int kCtas = RW == 8 ? 3 : 2;  // per SM
  static constexpr int kStages = WM == 4 ? 4 : RW == 8 ? 2 : 3;
  static constexpr int kStageBytes = 2 * kTile * HD;  // K rows, then V rows
  static constexpr int kRing = NS * kStages * kStageBytes;
  static constexpr int LDO = HD + 4;            // padded row of the join buffer
  static constexpr int kJoin = kWarps * RW * LDO * 4;
  static constexpr int kMain = kRing > kJoin ? kRing : kJoin;
  static constexpr int kSide = NS * kStages * 32;     // per stage: 4 scales and the block mask
  static constexpr int kQ = kRows * HD * 2;           // q as B fragments: [row / 8][dim / 16][lane] 8 bytes
  static constexpr int kSmem = kMain + kSide + kQ + kRows * 4;  // then what undoes each row's scaling
};

struct Segment {
  int b, rt, kvh;    // unit
  int tile0, tile1;  // position tiles
};

__device__ __forceinline__ int unit_cost(int n) { return n ? (n - 1) / kTile + 1 + kUnitCost : 0; }

// Attended positions of sequence b by its last real token of row tile rt; 0 where the tile has none.
template <int RT>
__device__ __forceinline__ int positions(const AttnParams& p, int b, int rt, int* news, int* len) {
  const int nn = p.new_lens ? min(p.new_lens[b], p.T) : p.T;
  const int ln = max(p.lens[b], 0);
  *news = nn;
  *len = ln;
  if (nn <= 0 || (long long)rt * RT >= (long long)nn * p.G) return 0;
  const int last = (int)min(((long long)rt * RT + RT - 1) / p.G, (long long)nn - 1);
  return (int)min((long long)ln + last + 1, (long long)p.max_pages * p.P);
}

template <int HD, int KIND, int RW, int WM>
__device__ __forceinline__ void run_segment(const AttnParams& p, const Segment& sg, bool whole, int slot, uint8_t* smem) {
  using S = Shape<HD, RW, WM>;
  constexpr int KT = HD / 16, MT = HD / 16, C = HD / 16, RT = S::kRows, LDO = S::LDO;
  constexpr int HH = RW / 8;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int grp = warp / WM, wm = warp % WM, r = lane >> 2, q4 = lane & 3;
  int news, len;
  const int n = positions<RT>(p, sg.b, sg.rt, &news, &len);
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + (uint32_t)(grp * S::kStages * S::kStageBytes);
  float* const side = reinterpret_cast<float*>(smem + S::kMain) + grp * S::kStages * 8;
  const int* trow = p.table + (long long)sg.b * p.ld_table;
  const int psh = p.P == 16 ? 4 : p.P == 32 ? 5 : 6;
  const long long page_codes = (long long)p.hkv * p.P * HD;
  const uint8_t* kbase = p.kv.k + (long long)sg.kvh * p.P * HD;
  const uint8_t* vbase = p.kv.v + (long long)sg.kvh * p.P * HD;

  auto group_sync = [&]() {
    if (WM == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + grp), "r"(32 * WM) : "memory");
  };
  // pages of a tile's two blocks of 16 positions, -1 past the unit's positions
  auto pages_of = [&](int tile, int& a, int& b) {
    const int t0 = tile * kTile;
    a = t0 < n ? valid_page(__ldg(trow + (t0 >> psh)), p.pages) : -1;
    b = a;
    if (p.P == 16 || t0 + 16 >= n) b = t0 + 16 < n ? valid_page(__ldg(trow + ((t0 + 16) >> psh)), p.pages) : -1;
  };
  constexpr int STEP = 32 * WM / C, PER = kTile / STEP;  // rows that the group copies at once, and how often
  const int gl = wm * 32 + lane, lrow = gl / C, lpiece = gl % C;
  const uint32_t kdst = ring + ((uint32_t)(lrow * HD + lpiece * 16) ^ k_key(lrow));
  const uint32_t vdst = ring + kTile * HD + ((uint32_t)(lrow * HD + lpiece * 16) ^ v_key<HD>(lrow));
  const int lsrc = lrow * HD + lpiece * 16;
  auto load = [&](int stage, int tile, int pa, int pb) {
    const int t0 = tile * kTile;
    const uint32_t ks = kdst + (uint32_t)(stage * S::kStageBytes), vs = vdst + (uint32_t)(stage * S::kStageBytes);
    // source of row 0 of the tile, were it in the page of block 0 or 1; absent blocks read as zeros
    const long long oa = max(pa, 0) * page_codes + (t0 & (p.P - 1)) * HD + lsrc;
    const long long ob = max(pb, 0) * page_codes + ((t0 + 16) & (p.P - 1)) * HD - 16 * HD + lsrc;
    const uint8_t *ka = kbase + oa, *kb = kbase + ob, *va = vbase + oa, *vb = vbase + ob;
    const uint32_t za = pa >= 0 ? 16u : 0u, zb = pb >= 0 ? 16u : 0u;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool second = STEP == 32 ? lrow >= 16 : i * STEP >= 16;
      const uint32_t z = second ? zb : za;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"((ks ^ k_key(i * STEP)) + i * STEP * HD), "l"((second ? kb : ka) + i * STEP * HD), "r"(z) : "memory");
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"((vs ^ v_key<HD>(i * STEP)) + i * STEP * HD), "l"((second ? vb : va) + i * STEP * HD), "r"(z) : "memory");
    }
    float* sd = side + stage * 8;
    if (gl < 4) {
      const int page = gl & 1 ? pb : pa;
      const float* src = (gl < 2 ? p.kv.ks : p.kv.vs) + (long long)max(page, 0) * p.hkv + sg.kvh;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"((uint32_t)__cvta_generic_to_shared(sd + gl)), "l"(src), "r"(page >= 0 ? 4u : 0u) : "memory");
    }
    if (gl == 4) sd[4] = __int_as_float((pa >= 0 ? 1 : 0) | (pb >= 0 ? 2 : 0));
  };
  // what this lane addresses for the matrix loads of stage 0
  const int krow = 4 * ((lane & 7) >> 1) + split_at(lane >> 4, lane & 1);
  const uint32_t kld = ring + ((uint32_t)(krow * HD + ((lane >> 3) & 1) * 16) ^ k_key(krow));
  const uint32_t vld = ring + kTile * HD + ((uint32_t)((lane & 15) * HD + (lane >> 4) * 16) ^ v_key<HD>(lane & 15));

  // q rows as the B operand, scaled by powers of two into f16; warps take 8 rows in turn
  uint2* const qs = reinterpret_cast<uint2*>(smem + S::kMain + S::kSide);
  float* const un = reinterpret_cast<float*>(smem + S::kMain + S::kSide + S::kQ);
  auto load_q = [&](int rg, uint2 (&w)[KT]) {
    const int row = sg.rt * RT + 8 * rg + r, t = row / p.G, g = row - t * p.G;
    const bool real = rg < RT / 8 && t < news;
    const uint16_t* src = p.q + ((long long)sg.b * p.T + (real ? t : 0)) * p.ld_q + (long long)(sg.kvh * p.G + (real ? g : 0)) * HD;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) w[kt] = real ? __ldg(reinterpret_cast<const uint2*>(src + kt * 16 + 4 * q4)) : make_uint2(0u, 0u);
  };
  auto store_q = [&](int rg, const uint2 (&w)[KT]) {
    float mx = 0.f;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
      mx = fmaxf(mx, fmaxf(fmaxf(fabsf(bf16_lo(w[kt].x)), fabsf(bf16_hi(w[kt].x))), fmaxf(fabsf(bf16_lo(w[kt].y)), fabsf(bf16_hi(w[kt].y)))));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    // 2^e with mx * 2^e in [2^14, 2^15), kept within normal floats
    const int e = min(max(14 + 127 - (int)(__float_as_uint(mx) >> 23), -112), 126);
    const float up = __uint_as_float((uint32_t)(e + 127) << 23);
    if (q4 == 0) un[8 * rg + r] = p.qscale * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const float x[4] = {bf16_lo(w[kt].x) * up, bf16_hi(w[kt].x) * up, bf16_lo(w[kt].y) * up, bf16_hi(w[kt].y) * up};
      qs[(rg * KT + kt) * 32 + lane] = make_uint2(pack_f16(x[k_at<KIND>(0, 0)], x[k_at<KIND>(0, 1)]),
                                                  pack_f16(x[k_at<KIND>(1, 0)], x[k_at<KIND>(1, 1)]));
    }
  };
  uint2 qw0[KT];  // this warp's first rows, asked for before the pages are looked up
  load_q(warp, qw0);

  // fill the ring
  const int first = sg.tile0 + grp;
#pragma unroll
  for (int s = 0; s < S::kStages - 1; ++s) {
    const int tile = first + s * S::NS;
    if (tile < sg.tile1) {
      int pa, pb;
      pages_of(tile, pa, pb);
      load(s, tile, pa, pb);
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  }
  int npa = -1, npb = -1;  // pages of the next tile to load
  if (first + (S::kStages - 1) * S::NS < sg.tile1) pages_of(first + (S::kStages - 1) * S::NS, npa, npb);

  if (warp < RT / 8) store_q(warp, qw0);
#pragma unroll
  for (int i = 1; i < (RT / 8 + kWarps - 1) / kWarps; ++i)
    if (i * kWarps + warp < RT / 8) {
      uint2 w[KT];
      load_q(i * kWarps + warp, w);
      store_q(i * kWarps + warp, w);
    }
  __syncthreads();
  const uint2* const qw = qs + wm * HH * KT * 32 + lane;
  float unscale[HH][2], m[HH][2], l[HH][2], vref = 1e-30f;  // of rows 8hh + 2 * q4 + e, as the scores below
  int lim[HH][2];                                           // positions those rows attend to
#pragma unroll
  for (int hh = 0; hh < HH; ++hh)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = wm * RW + 8 * hh + 2 * q4 + e, t = (sg.rt * RT + row) / p.G;
      unscale[hh][e] = un[row];
      lim[hh][e] = t < news ? (int)min((long long)len + t + 1, (long long)n) : n;  // rows that are not there compute something unread
      m[hh][e] = -INFINITY;
      l[hh][e] = 0.f;
    }
  const int lim_min = (int)min((long long)len + sg.rt * RT / p.G + 1, (long long)n);  // the unit's first row's

  float o[MT][HH][4];  // output, transposed: dims 16i + r (+ 8), rows 8hh + 2 * q4 (+ 1)
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int hh = 0; hh < HH; ++hh) o[i][hh][0] = o[i][hh][1] = o[i][hh][2] = o[i][hh][3] = 0.f;

  const Masks mk = p.masks;
  int stage = 0;
  for (int tile = first; tile < sg.tile1; tile += S::NS) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(S::kStages - 2) : "memory");
    group_sync();  // this stage has landed for the group, and the previous one is free
    const int ahead = tile + (S::kStages - 1) * S::NS;
    if (ahead < sg.tile1) {
      load(stage == 0 ? S::kStages - 1 : stage - 1, ahead, npa, npb);
      if (ahead + S::NS < sg.tile1) pages_of(ahead + S::NS, npa, npb);
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
    const uint32_t ks = kld + (uint32_t)(stage * S::kStageBytes), vs = vld + (uint32_t)(stage * S::kStageBytes);
    const float4 sc = *reinterpret_cast<const float4*>(side + stage * 8);  // K scales, V scales of the two blocks
    const int have = __float_as_int(side[stage * 8 + 4]);
    stage = stage + 1 == S::kStages ? 0 : stage + 1;

    // scores, transposed: s[j][hh][2h + e] is position 16j + 4 * (r / 2) + split_at(h, r % 2), row 8hh + 2 * q4 + e
    float s[2][HH][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int hh = 0; hh < HH; ++hh) s[j][hh][0] = s[j][hh][1] = s[j][hh][2] = s[j][hh][3] = 0.f;
#pragma unroll
    for (int c = 0; c < C; c += 2) {
      uint32_t w[2][4];  // pieces c, c + 1 of rows h = 0, then of rows h = 1
#pragma unroll
      for (int j = 0; j < 2; ++j) ldsm_x4((ks ^ (uint32_t)(c << 4)) + j * 16 * HD, w[j]);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint2 qf[HH];
#pragma unroll
        for (int hh = 0; hh < HH; ++hh) qf[hh] = qw[(hh * KT + c + x) * 32];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t a[4];
          to_f16<KIND>(mk, w[j][x], a[0], a[2]);
          to_f16<KIND>(mk, w[j][2 + x], a[1], a[3]);
#pragma unroll
          for (int hh = 0; hh < HH; ++hh) mma_f16(s[j][hh], a, qf[hh].x, qf[hh].y);
        }
      }
    }
    const int t0 = tile * kTile;
    bool grew = false;
#pragma unroll
    for (int hh = 0; hh < HH; ++hh)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][hh][e] *= unscale[hh][e & 1] * (j == 0 ? sc.x : sc.y);
    if (have != 3 || t0 + kTile > lim_min) {
#pragma unroll
      for (int hh = 0; hh < HH; ++hh)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!((have >> j) & 1) || t0 + 16 * j + 4 * (r >> 1) + split_at(e >> 1, r & 1) >= lim[hh][e & 1])
              s[j][hh][e] = -INFINITY;
    }
    float mn[HH][2];  // over this lane's positions
#pragma unroll
    for (int hh = 0; hh < HH; ++hh)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mn[hh][e] = fmaxf(fmaxf(s[0][hh][e], s[0][hh][2 + e]), fmaxf(s[1][hh][e], s[1][hh][2 + e]));
        grew |= mn[hh][e] > m[hh][e] + kSlack;
      }
    const float vmax = fmaxf(sc.z, sc.w);
    if (__any_sync(0xffffffffu, grew || vmax > vref)) {
      const float vr = vmax > vref ? vref / vmax : 1.f;
      vref = fmaxf(vref, vmax);
#pragma unroll
      for (int hh = 0; hh < HH; ++hh) {
        float av[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(m[hh][e], mn[hh][e]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          const float al = top == -INFINITY ? 0.f : ex2(m[hh][e] - top);
          m[hh][e] = top;
          l[hh][e] *= al;
          av[e] = al * vr;
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][hh][e] *= av[e & 1];
      }
    }
    const float vinv = 1.f / vref, vf[2] = {sc.z * vinv * v_unit<KIND>(), sc.w * vinv * v_unit<KIND>()};
#pragma unroll
    for (int hh = 0; hh < HH; ++hh)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float base = m[hh][e & 1] == -INFINITY ? 0.f : m[hh][e & 1];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float x = ex2(s[j][hh][e] - base);
          l[hh][e & 1] += x;
          s[j][hh][e] = x * vf[j];
        }
      }
    // V^T P^T, 16 positions at a time; each weight as a bf16 number and the rest of it
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t hi[HH][2], lo[HH][2];
#pragma unroll
      for (int hh = 0; hh < HH; ++hh)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float u = s[j][hh][2 * x], v = s[j][hh][2 * x + 1];
          const uint32_t w = pack_bf16(u, v);
          hi[hh][x] = transpose(w);
          lo[hh][x] = transpose(pack_bf16(u - bf16_lo(w), v - bf16_hi(w)));
        }
#pragma unroll
      for (int c = 0; c < C; c += 2) {
        uint32_t w[4];
        uint32_t a[2][4];
        ldsm_t8_x2((vs ^ (uint32_t)(c << 4)) + j * 16 * HD, w);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          to_bf16<KIND>(mk, w[2 * x], a[x][0], a[x][2]);
          to_bf16<KIND>(mk, w[2 * x + 1], a[x][1], a[x][3]);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int hh = 0; hh < HH; ++hh) mma_bf16(o[c + x][hh], a[x], hi[hh][0], hi[hh][1]);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int hh = 0; hh < HH; ++hh) mma_bf16(o[c + x][hh], a[x], lo[hh][0], lo[hh][1]);
      }
    }
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
#pragma unroll
  for (int hh = 0; hh < HH; ++hh)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[hh][e] += __shfl_xor_sync(0xffffffffu, l[hh][e], x);

  // join the warp groups: outputs and (max, sum) of every warp's rows
  __shared__ float2 wstat[kWarps][RW];
  __syncthreads();  // the ring is free
  float* po = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int hh = 0; hh < HH; ++hh) {
    float* dst = po + (warp * RW + 8 * hh + 2 * q4) * LDO + r;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      dst[16 * i] = o[i][hh][0] * v_rest<KIND>() * vref;
      dst[16 * i + LDO] = o[i][hh][1] * v_rest<KIND>() * vref;
      dst[16 * i + 8] = o[i][hh][2] * v_rest<KIND>() * vref;
      dst[16 * i + 8 + LDO] = o[i][hh][3] * v_rest<KIND>() * vref;
    }
    if (r == 0) {
      wstat[warp][8 * hh + 2 * q4] = make_float2(m[hh][0], l[hh][0]);
      wstat[warp][8 * hh + 2 * q4 + 1] = make_float2(m[hh][1], l[hh][1]);
    }
  }
  __syncthreads();
  const int rows = min(RT, news * p.G - sg.rt * RT);
  for (int i = tid; i < rows * (HD / 4); i += kThreads) {
    const int row = i / (HD / 4), c = i % (HD / 4), w0 = row / RW, rr = row % RW;
    float M = -INFINITY;
#pragma unroll
    for (int g = 0; g < S::NS; ++g) M = fmaxf(M, wstat[g * WM + w0][rr].x);
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int g = 0; g < S::NS; ++g) {
      const float2 st = wstat[g * WM + w0][rr];
      if (st.y == 0.f) continue;  // no position seen
      const float f = ex2(st.x - M);
      const float4 v = *reinterpret_cast<const float4*>(po + ((g * WM + w0) * RW + rr) * LDO + 4 * c);
      L = fmaf(f, st.y, L);
      acc.x = fmaf(f, v.x, acc.x);
      acc.y = fmaf(f, v.y, acc.y);
      acc.z = fmaf(f, v.z, acc.z);
      acc.w = fmaf(f, v.w, acc.w);
    }
    if (whole) {
      const float inv = L == 0.f ? 0.f : 1.f / L;
      const int grow = sg.rt * RT + row, t = grow / p.G, g = grow - t * p.G;
      uint16_t* dst = p.out + ((long long)sg.b * p.T + t) * p.ld_out + (long long)(sg.kvh * p.G + g) * HD + 4 * c;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
    } else {
      reinterpret_cast<float4*>(p.part)[((long long)slot * RT + row) * (HD / 4) + c] = acc;
      if (c == 0) p.stats[(long long)slot * RT + row] = make_float2(M, L);
    }
  }
  __syncthreads();  // the join buffer becomes the ring again
}

// Joins the runs c0 .. c1 of a unit, in order, by the last CTA that finished one.
template <int HD, int RW, int WM>
__device__ __forceinline__ void join_runs(const AttnParams& p, const Segment& sg, int c0, int c1, int slot0) {
  constexpr int RT = Shape<HD, RW, WM>::kRows;
  int news, len;
  positions<RT>(p, sg.b, sg.rt, &news, &len);
  const int rows = min(RT, news * p.G - sg.rt * RT);
  for (int i = threadIdx.x; i < rows * (HD / 4); i += kThreads) {
    const int row = i / (HD / 4), c = i % (HD / 4);
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int N = 8;  // runs whose loads are in flight together
    for (int k0 = c0; k0 <= c1; k0 += N) {
      float2 st[N];
      float4 v[N];
#pragma unroll
      for (int x = 0; x < N; ++x) {
        st[x] = make_float2(0.f, 0.f);
        if (k0 + x <= c1) {
          const long long at = (long long)(k0 + x == c0 ? slot0 : 2 * (k0 + x)) * RT + row;
          st[x] = __ldcg(p.stats + at);
          v[x] = __ldcg(reinterpret_cast<const float4*>(p.part) + at * (HD / 4) + c);
        }
      }
#pragma unroll
      for (int x = 0; x < N; ++x) {
        if (st[x].y == 0.f) continue;  // no position seen
        const float mn = fmaxf(M, st[x].x), a = ex2(M - mn), f = ex2(st[x].x - mn);
        M = mn;
        L = fmaf(L, a, f * st[x].y);
        acc.x = fmaf(acc.x, a, f * v[x].x);
        acc.y = fmaf(acc.y, a, f * v[x].y);
        acc.z = fmaf(acc.z, a, f * v[x].z);
        acc.w = fmaf(acc.w, a, f * v[x].w);
      }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int grow = sg.rt * RT + row, t = grow / p.G, g = grow - t * p.G;
    uint16_t* dst = p.out + ((long long)sg.b * p.T + t) * p.ld_out + (long long)(sg.kvh * p.G + g) * HD + 4 * c;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
  }
}

template <int HD, int KIND, int RW, int WM>
__global__ void __launch_bounds__(kThreads, Shape<HD, RW, WM>::kCtas) kv8_attention_kernel(const __grid_constant__ AttnParams p) {
  using S = Shape<HD, RW, WM>;
  constexpr int RT = S::kRows;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ unsigned prefix[kMaxEntries + 1];  // cost of one kv head before each entry
  __shared__ unsigned wsum[kWarps];
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  chain();
  // a run of position tiles (with kUnitCost more before each unit's), or every gridDim-th unit
  unsigned per = 0, at = blockIdx.x, end = p.units;
  int e = 0, kvh = 0;
  if (p.balanced) {
    // cost of each entry and their running sum
    const int ne = p.B * p.row_tiles, each = (ne + kThreads - 1) / kThreads, e0 = min(tid * each, ne), e1 = min(e0 + each, ne);
    unsigned mine = 0;
    for (int i = e0; i < e1; ++i) {
      int news, len;
      mine += unit_cost(positions<RT>(p, i / p.row_tiles, i % p.row_tiles, &news, &len));
    }
    unsigned inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    unsigned sum = inc - mine;
    for (int w = 0; w < warp; ++w) sum += wsum[w];
    for (int i = e0; i < e1; ++i) {
      int news, len;
      prefix[i] = sum;
      sum += unit_cost(positions<RT>(p, i / p.row_tiles, i % p.row_tiles, &news, &len));
    }
    if (e1 == ne && e0 < e1) prefix[ne] = sum;
    __syncthreads();
    const unsigned total = prefix[ne] * p.hkv;
    per = max((total + gridDim.x - 1) / gridDim.x, (unsigned)kMinTiles);
    // the entry that holds x < total: the last with hkv * prefix <= x
    auto entry_of = [&](unsigned x) {
      int lo = 0, hi = ne - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] * p.hkv <= x) lo = mid;
        else hi = mid - 1;
      }
      return lo;
    };
    // run boundaries inside a short unit move to its nearer end
    auto boundary = [&](unsigned i) {
      const unsigned x = i * per;
      if (x >= total) return total;
      const int b = entry_of(x);
      const unsigned cost = prefix[b + 1] - prefix[b], into = (x - prefix[b] * p.hkv) % cost;
      return cost > kWholeCost ? x : 2 * into < cost ? x - into : x - into + cost;
    };
    at = boundary(blockIdx.x);
    end = boundary(blockIdx.x + 1);
    if (at < end) {
      e = entry_of(at);
      kvh = (int)((at - prefix[e] * p.hkv) / (prefix[e + 1] - prefix[e]));
    }
  }
  const unsigned begin = at;
  while (at < end) {
    Segment sg;
    unsigned r0 = 0, u1 = 0;  // the unit's first tile and its end
    bool whole = true, leads = false;
    if (p.balanced) {
      const unsigned cost = prefix[e + 1] - prefix[e];
      if (kvh == p.hkv || cost == 0) {
        ++e;
        kvh = 0;
        continue;
      }
      r0 = prefix[e] * p.hkv + kvh * cost + kUnitCost;
      u1 = r0 + cost - kUnitCost;
      const unsigned stop = min(end, u1), s0 = max(at, r0);
      at = stop;
      sg.kvh = kvh++;
      if (s0 >= stop) continue;
      sg.tile0 = (int)(s0 - r0);
      sg.tile1 = (int)(stop - r0);
      whole = s0 == r0 && stop == u1;
      leads = s0 == begin;
    } else {
      e = (int)(at / p.hkv);
      sg.kvh = (int)(at % p.hkv);
      at = at + gridDim.x < at ? end : at + gridDim.x;
    }
    sg.b = e / p.row_tiles;
    sg.rt = e % p.row_tiles;
    if (!p.balanced) {
      int news, len;
      const int n = positions<RT>(p, sg.b, sg.rt, &news, &len);
      if (n == 0) continue;
      sg.tile0 = 0;
      sg.tile1 = (n - 1) / kTile + 1;
    }
    run_segment<HD, KIND, RW, WM>(p, sg, whole, 2 * blockIdx.x + (leads ? 0 : 1), smem);
    if (!whole) {
      const int c0 = (int)(r0 / per), c1 = (int)((u1 - 1) / per);
      if (tid == 0) {  // the other threads' stores came before the barrier that ended run_segment
        unsigned before;
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(p.counter + c0) : "memory");
        last = before == (unsigned)(c1 - c0);
        if (last) p.counter[c0] = 0u;  // ready for the next call
      }
      __syncthreads();
      if (last) join_runs<HD, RW, WM>(p, sg, c0, c1, 2 * c0 + (r0 == c0 * per ? 0 : 1));
      __syncthreads();
    }
  }
  // rows without a position are zeros: each CTA takes its share of the batch's rows
  for (long long m = blockIdx.x; m < (long long)p.B * p.T; m += gridDim.x) {
    const int b = (int)(m / p.T), t = (int)(m - (long long)b * p.T);
    const int nn = p.new_lens ? p.new_lens[b] : p.T;
    if (t >= nn)
      for (int i = tid; i < p.hq * HD / 8; i += kThreads)
        *reinterpret_cast<uint4*>(p.out + m * p.ld_out + 8 * i) = make_uint4(0u, 0u, 0u, 0u);
  }
}

// Row tile of a call: the smallest of 8, 16, 24, 32, 48, 64 that holds the rows
// of a kv head; beyond, 64 or 96, whichever pads them less.
int row_tile(int64_t T, int G) {
  const int64_t rows = T * G;
  for (int t : {8, 16, 24, 32, 48, 64})
    if (rows <= t) return t;
  return (rows + 95) / 96 * 96 <= (rows + 63) / 64 * 64 ? 96 : 64;
}

// CTAs that fill the GPU once.
int grid_of(int rows) { return sm_count() * (rows == 8 ? 3 : 2); }

// The counters have one place whatever the row tile, so that calls of different
// tokens per sequence find them at zero where the others left them.
size_t counter_bytes() { return ((size_t)3 * sm_count() * sizeof(unsigned) + 255) & ~(size_t)255; }

template <int HD, int KIND, int RW, int WM>
int launch(const AttnParams& p, int grid, cudaStream_t st) {
  constexpr int smem = Shape<HD, RW, WM>::kSmem;
  static_assert((smem + 6 * 1024) * Shape<HD, RW, WM>::kCtas <= 227 * 1024, "resident CTAs");
  auto kern = kv8_attention_kernel<HD, KIND, RW, WM>;
  static std::atomic<uint64_t> allowed{0};  // devices where the kernel may use its shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return WAL_ERR_CUDA;
  if (!(allowed.load(std::memory_order_relaxed) >> dev & 1)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return WAL_ERR_CUDA;
    allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  return launch_chain(kern, dim3((unsigned)grid), kThreads, smem, st, p);
}

template <int HD, int KIND>
int launch_rows(const AttnParams& p, int rows, int grid, cudaStream_t st) {
  switch (rows) {
    case 8: return launch<HD, KIND, 8, 1>(p, grid, st);
    case 16: return launch<HD, KIND, 16, 1>(p, grid, st);
    case 24: return launch<HD, KIND, 24, 1>(p, grid, st);
    case 32: return launch<HD, KIND, 16, 2>(p, grid, st);
    case 48: return launch<HD, KIND, 24, 2>(p, grid, st);
    case 64: return launch<HD, KIND, 16, 4>(p, grid, st);
    default: return launch<HD, KIND, 24, 4>(p, grid, st);
  }
}

}  // namespace

extern "C" {

size_t wal_kv8_attention_workspace(const wal_kv8_cache* cache, int64_t B, int64_t T, int32_t hq) {
  if (!cache || cache->kv_heads <= 0 || B <= 0 || T <= 0 || hq <= 0 || hq % cache->kv_heads || T > 0x7fffffff) return 0;
  int64_t rows = row_tile(T, hq / cache->kv_heads);
  if (rows == 64 && T * (hq / cache->kv_heads) > 64) rows = 96;  // never less for more tokens
  const int grid = grid_of((int)rows);
  return counter_bytes() + (size_t)grid * 2 * rows * (cache->head_dim * sizeof(float) + sizeof(float2));
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
  if (B > 0x7fffffff || T > 0x7fffffff || max_pages > (0x7fffffff - kTile) / cache->page_size || B * T > 0x7fffffff / hq) return WAL_ERR_SHAPE;
  if (ld_q < (int64_t)hq * hd || ld_out < (int64_t)hq * hd) return WAL_ERR_SHAPE;
  if (((uintptr_t)q & 15) || ((uintptr_t)out & 15) || ((uintptr_t)workspace & 255) || (ld_q % 8) || (ld_out % 8)) return WAL_ERR_ALIGNMENT;
  if (workspace_bytes < wal_kv8_attention_workspace(cache, B, T, hq)) return WAL_ERR_BUFFER_TOO_SMALL;
  AttnParams p = {};
  p.q = q;
  p.ld_q = ld_q;
  p.kv = layer_view(*cache, layer);
  p.B = (int)B;
  p.T = (int)T;
  p.hq = hq;
  p.hkv = cache->kv_heads;
  p.G = hq / cache->kv_heads;
  p.P = cache->page_size;
  p.pages = (int)cache->num_pages;
  p.max_pages = (int)max_pages;
  const int rows = row_tile(T, p.G), grid = grid_of(rows);
  p.row_tiles = (int)((T * p.G + rows - 1) / rows);
  p.table = table;
  p.ld_table = ld_table;
  p.lens = lens;
  p.new_lens = new_lens;
  p.qscale = scale * 1.4426950408889634f;  // log2(e)
  p.out = out;
  p.ld_out = ld_out;
  // the sums of costs fit 32 bits, whatever the lengths
  if (B * p.row_tiles > 0xffffffffLL / p.hkv) return WAL_ERR_SHAPE;
  p.units = (unsigned)(B * p.row_tiles * p.hkv);
  p.balanced = B * p.row_tiles <= kMaxEntries &&
               (long long)p.units * (max_pages * p.P / kTile + 1 + kUnitCost) + (long long)grid * kMinTiles * 2 < (1LL << 31);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.counter = reinterpret_cast<unsigned*>(ws);
  p.part = reinterpret_cast<float*>(ws + counter_bytes());
  p.stats = reinterpret_cast<float2*>(p.part + (size_t)grid * 2 * rows * hd);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (hd == 128)
    return cache->kind == WAL_KV_INT8 ? launch_rows<128, WAL_KV_INT8>(p, rows, grid, s) : launch_rows<128, WAL_KV_E4M3>(p, rows, grid, s);
  return cache->kind == WAL_KV_INT8 ? launch_rows<64, WAL_KV_INT8>(p, rows, grid, s) : launch_rows<64, WAL_KV_E4M3>(p, rows, grid, s);
}

}  // extern "C"
