// kv8_attention.cu -- attention of a few new tokens per sequence over the paged 8-bit cache.
//
// Maths, per query row r (a new token and a query head) over the cached tokens j it sees:
//   s_j = sm_scale (q . k8_j) ks_j,   o = sum_j e^{s_j} vs_j v8_j / sum_j e^{s_j}
// with k8, v8 the cached bytes' values and ks, vs the scales of token j's (page, head).
//
// Bound: HBM, the cache's bytes (4 heads_q / heads_kv flops per byte).  So up to 16 rows that read the same keys
// and values -- the tokens and heads of a group -- share one pass over them (more rows are units of their own, each with
// its pass: 20 sequences of up to 9000 tokens, Hq 32 Hkv 4 D 128, 16 rows of two queries 35 us, 32 of four 61, 128 of
// sixteen 212), and the work is cut along the sequences so that every SM streams until the end:
//   * a unit is (sequence, key/value head, tile of 8 or 16 rows); its tokens come in tiles of 16 (D 256), 32 or
//     64 (D 64, 8 rows).  All units' tiles laid end to end are cut into equal ranges, one per CTA of a grid that fills the GPU once;
//     lengths are read on the device, so the launch does not depend on them.  A unit inside one range is written
//     directly; a unit cut by range borders leaves normalised partial rows with their maximum and sum, and a second
//     kernel joins them in the order of the CTAs (launched to start as the first drains).  Results do not depend on
//     timing.  Where the table has room for short sequences only, each unit has a CTA of its own instead and the
//     second kernel falls away (one sequence of 129 tokens: 6.5 to 7.1 us; 2400 units of up to 1024: 89 -> 80).  The same
//     sequences with a wide table pay for plan and join (129 tokens 9.7 us; 16 x 1031, four queries 8.8 -> 12), the more the
//     larger the batch, since every CTA forms the plan (8192 sequences of 512, Hkv 1, D 128: 210 -> 430).
//   * a CTA's 4, 8 or 12 warps take its range's tiles in turn, each with a ring of its own in shared memory (cp.async,
//     192 KB per SM in flight) that is filled ahead over unit borders, so that a change of unit costs no memory latency.  Only changes of unit have barriers; there is no wait on another CTA.
//   * scores S^T = K Q^T and outputs O^T = V^T P^T are m16n8k16 products with the cache's bytes as the 16-row
//     operand, widened to fp16 in registers (exact) -- the order of the head dimension inside a product is free, so a
//     lane's 16 bytes of a key are its fragments as they lie.  Accumulation is fp32.  tcgen05 products would take
//     128 rows of bytes for 8 to 16 query rows and need the bytes in one 8-bit type with the weights, which 8 bits do
//     not hold; the e4m3 form of this product runs on the same pipe with the same widening inside (it measured 5 % slower).
// What it measured (B200, device time): Hq 32 Hkv 8 D 128, 64 sequences of 1024 to 4096 tokens 61.5 us, 5.5 TB/s (the same
// copies without the products 59 us at a time when the whole took 64); Hq 16 Hkv 2 D 256, 16 sequences of up to 65536 tokens
// 112 to 114 us, 5.7 TB/s; one of 65536 20.5 to 20.8 us.  The SMs' shares of the bandwidth differ (equal ranges ended after
// 86 to 110 us of those), but short ranges drawn as SMs got done cost more in changes of unit than they evened out.  16 rows and
// D >= 128 are bound by eight warps' latency instead: 20 sequences of up to 9000 tokens, Hq 32 Hkv 4, two queries, 35 us,
// 2.9 TB/s.  The figures beside the choices below (tiles, warps, layouts, joins) were taken before each row had its own
// reference (last paragraph), which adds the same to both sides.
//
// Number formats.  q rows enter fp16 after scaling by a power of two that brings their largest element to
// [2^14, 2^15): exact for elements down to 2^-28 of it (bf16 has 8 bits, fp16 11).  A weight enters with its scale, as
// 2^14 e^{s_j} vs_j / 2^mv rounded to fp16 (half a step is 2^-11), mv the largest s_j + log2 vs_j (s in base 2) the row has met:
// the products fill fp16's range whatever the scales are, and only what is under 2^-39 of the row's largest e^{s_j} vs_j
// vanishes.  (One reference for all rows, the largest vs_j loaded, would let a block of little or no weight take the
// others' bits; a reference per row costs 8 rows up to 2 %, 16 rows 3 to 11 %: 20 sequences of up to 9000 tokens, Hq 32 Hkv 4
// D 128, two queries, 33.0 -> 35.1 us.)  Maxima, sums and outputs are fp32; weights under 2^-140 of the largest are zero.
#include "kv8_common.cuh"

#include <algorithm>
#include <cmath>

namespace tokmix {
namespace kv8 {

constexpr int kMaxTokens = 16;
constexpr int kMaxBatch = 8192;  // the plan keeps batch + 1 words in shared memory
constexpr float kShift = 14.0f;  // weights are held times 2^14
// a little under 126, so that 2^-kRise stays a normal number when the score it is added to rounds the sum up; a weight times a
// scale of up to 2^127.9 is then within fp16
constexpr float kRise = 125.9375f;
constexpr float kSpan = 112.0f;  // a row's accumulators are held times 2^112 / (its largest weight) at most
constexpr int kJoinThreads = 256;
constexpr int kMaxCtas = 512;  // at most 3 per SM

template <int D, int NT>
struct Shape {
  static constexpr int kTok = D == 256 ? 16 : D == 64 && NT == 1 ? 64 : 32;  // tokens per tile: 8 KB, 4 KB (D 64, 16 rows)
  static constexpr int kMt = kTok / 16;       // 16-token subtiles (a page holds whole ones)
  static constexpr int kRows = 8 * NT;        // query rows per unit
  static constexpr int kQStride = D + 8;      // halves between rows of q in shared memory (conflict-free 16-byte reads)
  static constexpr int kStageBytes = 2 * kTok * D;              // a tile's keys and values
  // 168 or 255 registers a thread: 16 rows of D 64 fit 168 (64 sequences of up to 2000 tokens 44.9 -> 41.9 us), of D 128 do
  // not (20 sequences of up to 9000 tokens, two queries: 33 us, with twelve warps 39 to 43)
  static constexpr int kWarpsPerSm = NT == 1 || D == 64 ? 12 : 8;
  static constexpr int kStages = 196608 / kWarpsPerSm / kStageBytes;  // 192 KB of tiles per SM
  __host__ __device__ static constexpr int smem_bytes(int warps) { return warps * kStages * (kStageBytes + 8 * kMt) + kRows * kQStride * 2; }
  static_assert(8 * D * 4 <= kStageBytes, "eight partial rows fit a stage");
  static_assert(kWarpsPerSm <= 16, "a row's warps are joined by 16 lanes");
};

struct AttnParams {
  View c;
  const void* q;
  long long q_sb, q_st, q_sh;
  void* out;
  float* lse;
  float* part_o;    // [2 grid][rows][D] normalised partial rows
  float2* part_ml;  // [2 grid][rows] (maximum, sum)
  int tokens, hq, group;
  int bf16;
  float scale_log2;  // sm_scale * log2(e)
  int grid;          // CTAs of the attention kernel
  int min_tiles;     // a CTA's range is at least this long
  int row_lines, table_lines;  // 128-byte lines of a table row, of the table
  int single;                  // a CTA per unit: none is cut
  uint32_t* status;
};

// ------------------------------------------------------------------------------------ the plan
// What a change of unit costs a CTA, in tiles (its warps end at different times, join, and start anew): ranges that count it
// end together (128 sequences of up to 1024 tokens, Hq 32 Hkv 8 D 128: 0 53.3 us, 4 47.8, 8 45.3, 12 44.0, 16 43.7, 24 43.9;
// with tiles of 64 tokens, 32 sequences of up to 2500, Hq 32 Hkv 8 D 64: 4 24.0 us, 8 23.0, 12 24.3).
template <int TOK>
constexpr int kUnitCost = TOK == 64 ? 8 : 12;

struct Unit {
  int tiles;      // token tiles of each of the sequence's units
  int row_tiles;  // row tiles per key/value head
  int length;     // of a unit on the line: kUnitCost places without a tile, then its tiles
};

template <int TOK, int ROWS>
__device__ __forceinline__ Unit unit_of(const AttnParams& p, const Seq& s) {
  Unit u;
  u.tiles = (s.end + TOK - 1) / TOK;
  u.row_tiles = ((s.end - s.start) * p.group + ROWS - 1) / ROWS;
  u.length = u.tiles + kUnitCost<TOK>;
  return u;
}

// prefix[b] = places on the line of the sequences before b, prefix[batch] = all; every thread calls.
template <int TOK, int ROWS, int THREADS>
__device__ __forceinline__ void make_plan(const AttnParams& p, uint32_t* prefix, uint32_t* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t carry = 0;
  for (int b0 = 0; b0 < p.c.batch; b0 += THREADS) {
    const int b = b0 + threadIdx.x;
    uint32_t n = 0;
    if (b < p.c.batch) {
      const Seq s = load_seq(p.c, b, p.tokens);
      const Unit u = unit_of<TOK, ROWS>(p, s);
      n = static_cast<uint32_t>(u.length) * u.row_tiles * p.c.hkv;
      if (!s.ok && blockIdx.x == 0) report_bad(p.status);
    }
    uint32_t sum = n;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, sum, off);
      if (lane >= off) sum += up;
    }
    if (lane == 31) scratch[warp] = sum;
    __syncthreads();
    uint32_t before = carry;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += scratch[w];
      carry += scratch[w];
    }
    if (b < p.c.batch) prefix[b] = before + sum - n;
    __syncthreads();
  }
  if (threadIdx.x == 0) prefix[p.c.batch] = carry;
  __syncthreads();
}

// CTAs that take part: none has an empty range (it may lie in a unit's places without a tile)
__device__ __forceinline__ uint32_t active_ctas(const AttnParams& p, uint32_t total) {
  return min(static_cast<uint32_t>(p.grid), max(1u, total / p.min_tiles));
}
__device__ __forceinline__ uint32_t range_begin(uint32_t cta, uint32_t total, uint32_t ctas) {
  return static_cast<uint32_t>(static_cast<unsigned long long>(cta) * total / ctas);
}
// the CTA whose range holds tile t: the last one with range_begin <= t
__device__ __forceinline__ uint32_t cta_of(uint32_t t, uint32_t total, uint32_t ctas) {
  return static_cast<uint32_t>(((static_cast<unsigned long long>(t) + 1) * ctas - 1) / total);
}

// ------------------------------------------------------------------------------------ small pieces
// four bytes -> four halves (two registers), exact
template <bool E4M3>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (E4M3) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
  } else {  // 1024 + (b + 128) is the half 0x64uu with u = b + 128; minus 1152
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const uint32_t k = 0x64806480u;
    const __half2 ra = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&k));
    const __half2 rb = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&k));
    lo = *reinterpret_cast<const uint32_t*>(&ra);
    hi = *reinterpret_cast<const uint32_t*>(&rb);
  }
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// transposes an 8x8 matrix of halves held as the rows of a fragment
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// log2 |x|; -infinity for 0 and subnormals
__device__ __forceinline__ float lg2_abs(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fabsf(x)));
  return y;
}

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float nan_f() { return __uint_as_float(0x7fc00000u); }

// 0x80 in every byte of four e4m3 ones that is NaN (0x7f, 0xff)
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

__device__ __forceinline__ void store_out4(const AttnParams& p, size_t at, const float (&o)[4]) {
  uint2 w;
  if (p.bf16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(o[0], o[1]), b = __floats2bfloat162_rn(o[2], o[3]);
    w = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) = w;
  } else {
    w = make_uint2(half2_bits(o[0], o[1]), half2_bits(o[2], o[3]));
    *reinterpret_cast<uint2*>(static_cast<__half*>(p.out) + at) = w;
  }
}

// m and sum of a row are in the base-2 domain with weights times 2^14
__device__ __forceinline__ float lse_of(float m, float sum) {
  return sum == 0.0f ? -INFINITY : (m - kShift + log2f(sum)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------------------------ attention
// One unit's share of a CTA's range
struct Segment {
  Seq s;
  int b, kvh, row0, rows_valid;  // rows row0 .. of the rows_valid of the sequence's key/value head
  int t0, t1;                    // token tiles
  bool whole;                    // all of the unit
};

// The tiles of a CTA's range in order, unit by unit
template <int TOK, int ROWS>
struct Walk {
  uint32_t pos, stop;
  int b;
  int kvh, row0;  // single: the CTA's one unit, as a range of one
  __device__ __forceinline__ bool next(const AttnParams& p, const uint32_t* prefix, Segment& n) {
    while (pos < stop) {
      if (!p.single)
        while (prefix[b + 1] <= pos) ++b;
      n.b = b;
      n.s = load_seq(p.c, b, p.tokens);
      n.rows_valid = (n.s.end - n.s.start) * p.group;
      const Unit u = unit_of<TOK, ROWS>(p, n.s);
      if (p.single) {
        n.t0 = 0;
        n.t1 = u.tiles;
        n.kvh = kvh;
        n.row0 = row0;
        n.whole = true;
        pos = stop;
        return true;
      }
      const int off = static_cast<int>(pos - prefix[b]);
      const int ui = off / u.length;
      const int from = off - ui * u.length, to = min(u.length, from + static_cast<int>(stop - pos));
      pos += to - from;
      if (to <= kUnitCost<TOK>) continue;  // the range ends before the unit's first tile
      n.t0 = max(from - kUnitCost<TOK>, 0);
      n.t1 = to - kUnitCost<TOK>;
      n.kvh = ui / u.row_tiles;
      n.row0 = (ui - n.kvh * u.row_tiles) * ROWS;
      n.whole = n.t0 == 0 && n.t1 == u.tiles;
      return true;
    }
    return false;
  }
};

// Byte offset of 16-byte chunk c of token row r in a tile in shared memory: rows of D bytes, chunks permuted inside each
// 128-byte line so that the reads below meet every bank once.  D >= 128: c ^ (r % 8).  D = 64 (two rows a line):
// line chunk 4 (r % 2) + c, ^ 2 ((r / 2) % 4).
template <int D>
__device__ __forceinline__ int tile_chunk(int r, int c) {
  if constexpr (D == 64) return (r >> 1) * 128 + ((((r & 1) << 2 | c) ^ (((r >> 1) & 3) << 1)) << 4);
  return r * D + ((c ^ (r & 7)) << 4);
}

// 16-byte chunk of a partial row in shared memory: spread so that the four rows a store instruction meets fall into
// different banks (a store's eight lanes hold rows 2 cq + e and chunks 4 g + x, or 2 g + x at D = 64)
template <int D>
__device__ __forceinline__ int merge_chunk(int row, int chunk) {
  const int cq = (row >> 1) & 3;
  return chunk ^ (D == 64 ? (cq & 1) | ((cq >> 1) << 2) : cq);
}

__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// the same, or zeros if !live (nothing is read then)
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const uint8_t* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

template <int D, bool E4M3, int NT, int W>
__global__ void __launch_bounds__(32 * W, Shape<D, NT>::kWarpsPerSm / W) attn_kernel(const AttnParams p) {
  using S = Shape<D, NT>;
  constexpr int TOK = S::kTok, MT = S::kMt, ROWS = S::kRows, J = D / 64, STAGES = S::kStages;
  constexpr int kVec = D / 8;  // 16-byte vectors of a query row
  constexpr int kThreads = 32 * W;
  constexpr int kQv = (ROWS * kVec + kThreads - 1) / kThreads;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem + (threadIdx.x >> 5) * STAGES * S::kStageBytes;                 // this warp's [stage][keys, values]
  float* scales = reinterpret_cast<float*>(smem + W * STAGES * S::kStageBytes) + (threadIdx.x >> 5) * STAGES * 2 * MT;
  __half* qs = reinterpret_cast<__half*>(smem + W * STAGES * (S::kStageBytes + 8 * MT));  // [row][kQStride]
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem + S::smem_bytes(W));
  __shared__ float row_factor[ROWS], row_top[ROWS], row_sum[ROWS], row_up[ROWS], warp_m[W][ROWS], warp_l[W][ROWS], warp_mv[W][ROWS];
  __shared__ int warp_at[W];  // where in `smem` a warp's partial rows lie
  // each warp's lane 0 alone; reported at the end (beside the loads: 400 sequences of up to 640, Hkv 8, D 128, 78.2 -> 79.3 us)
  __shared__ int met_bad_page[W];
  __shared__ uint32_t scratch[W];

  const View& c = p.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, cq = lane & 3;

  wait_previous_kernels();
  asm volatile("griddepcontrol.launch_dependents;");  // the join kernel, which reads the lengths before it waits
  if (blockIdx.x * kThreads + threadIdx.x < p.table_lines) {  // the table, read behind the plan, on its way to L2
    const int line = blockIdx.x * kThreads + threadIdx.x, row = line / p.row_lines;
    asm volatile("prefetch.global.L2 [%0];" ::"l"(c.table + row * c.table_stride + (line - row * p.row_lines) * 32));
  }
  Walk<TOK, ROWS> walk;
  if (p.single) {  // short sequences: a CTA per unit, no plan and nothing to join
    const int row_tiles = (p.tokens * p.group + ROWS - 1) / ROWS;
    walk.b = blockIdx.x / (row_tiles * c.hkv);
    const int ui = blockIdx.x - walk.b * row_tiles * c.hkv;
    walk.kvh = ui / row_tiles;
    walk.row0 = (ui - walk.kvh * row_tiles) * ROWS;
    walk.pos = 0;
    walk.stop = 1;
    const Seq s = load_seq(c, walk.b, p.tokens);
    if (!s.ok && threadIdx.x == 0) report_bad(p.status);
    const int seen = max(walk.row0, (s.end - s.start) * p.group), last = min(walk.row0 + ROWS, p.tokens * p.group);
    const float f = s.ok ? 0.0f : nan_f();  // rows that see nothing
    const float o[4] = {f, f, f, f};
    for (int v = threadIdx.x; v < (last - seen) * (D / 4); v += kThreads) {
      const int row = seen + v / (D / 4), x = v % (D / 4);
      const int i = row / p.group, h = walk.kvh * p.group + row - i * p.group;
      const size_t orow = (static_cast<size_t>(walk.b) * p.tokens + i) * p.hq + h;
      store_out4(p, orow * D + 4 * x, o);
      if (p.lse != nullptr && x == 0) p.lse[orow] = s.ok ? -INFINITY : f;
    }
    if (seen == walk.row0) return;
  } else {
    make_plan<TOK, ROWS, kThreads>(p, prefix, scratch);
    const uint32_t total = prefix[c.batch];
    if (total == 0) return;
    const uint32_t ctas = active_ctas(p, total);
    if (blockIdx.x >= ctas) return;
    walk.pos = range_begin(blockIdx.x, total, ctas);
    walk.stop = range_begin(blockIdx.x + 1, total, ctas);
    walk.b = 0;
    for (int hi = c.batch; hi - walk.b > 1;) {  // the last sequence with prefix <= pos
      const int mid = (walk.b + hi) >> 1;
      if (prefix[mid] <= walk.pos) walk.b = mid; else hi = mid;
    }
  }

  // byte offsets inside a tile: this lane's share of a copy, its keys, its values
  constexpr int kCopies = D == 64 ? 1 : D == 128 ? 2 : 4;
  uint32_t cp_off[kCopies], k_off[2], v_off[2];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) cp_off[i] = tile_chunk<D>((i * 32 + lane) / (D / 16), lane % (D / 16)) - i * 512;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    k_off[i] = tile_chunk<D>(g, D == 64 ? cq : 2 * cq + i);
    v_off[i] = D == 64 ? tile_chunk<D>(2 * cq + i, g >> 1) + (g & 1) * 8 : tile_chunk<D>(2 * cq + i, g);
  }

  // ---- the loads run ahead of the products by up to STAGES tiles, across units; table entries by one more
  Walk<TOK, ROWS> ahead = walk;
  Segment ld{};         // unit of the next tile to load
  int ld_t = 0;         // that tile
  bool ld_live;         // false: no tile is left
  int pid[MT];          // its pages
  int ld_stage = 0;
  const uint8_t *ld_k = nullptr, *ld_v = nullptr;  // its head in page 0, this lane's 16 bytes
  auto find_tile = [&]() {
    while (ld_live && ld_t >= ld.t1) {
      ld_live = ahead.next(p, prefix, ld);
      if (ld_live) {
        ld_t = ld.t0 + warp;
        ld_k = c.k + ld.kvh * c.k_head_stride + lane * 16;
        ld_v = c.v + ld.kvh * c.v_head_stride + lane * 16;
      }
    }
    if (ld_live) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)  // behind the sequence's end: its last page
        pid[mt] = __ldg(c.table + ld.b * c.table_stride + (min(ld_t * TOK + mt * 16, ld.s.end - 1) >> c.page_shift));
    }
  };
  auto load_tile = [&]() {
    if (ld_live) {
      const uint32_t dst0 = smem_addr(ring + ld_stage * S::kStageBytes);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int tok = ld_t * TOK + mt * 16;
        const bool good = static_cast<unsigned>(pid[mt]) < static_cast<unsigned>(c.num_pages);
        const uint32_t pg = good ? pid[mt] : 0;
        const int slot = (tok & (c.page - 1)) * D;
        const uint8_t* ksrc = ld_k + static_cast<unsigned long long>(pg) * static_cast<uint32_t>(c.k_page_stride) + slot;
        const uint8_t* vsrc = ld_v + static_cast<unsigned long long>(pg) * static_cast<uint32_t>(c.v_page_stride) + slot;
        const int rows = good ? ld.s.end - tok : 0;  // token rows to read; zeros behind them
        if (rows >= 16) {
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            const uint32_t dst = dst0 + mt * 16 * D + i * 512 + cp_off[i % kCopies];
            copy16(dst, ksrc + i * 512);
            copy16(dst + TOK * D, vsrc + i * 512);
          }
        } else {
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            const int r = (i * 32 + lane) / (D / 16);
            const uint32_t dst = dst0 + mt * 16 * D + i * 512 + cp_off[i % kCopies];
            copy16_or_zero(dst, ksrc + i * 512, r < rows);
            copy16_or_zero(dst + TOK * D, vsrc + i * 512, r < rows);
          }
        }
        float* sc = scales + ld_stage * 2 * MT + mt;
        if (good) {
          if (lane < 2) copy4(smem_addr(sc + lane * MT), (lane == 0 ? c.k_scale : c.v_scale) + static_cast<unsigned long long>(pg) * static_cast<uint32_t>(c.hkv) + ld.kvh);
        } else if (lane < 2) {  // NaN scores for the rows that see it
          sc[lane * MT] = lane == 0 && tok < ld.s.end ? nan_f() : 0.0f;
          if (lane == 0 && tok < ld.s.end) met_bad_page[warp] = 1;
        }
      }
      ld_t += W;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");  // an empty group too: the waits count groups
    ld_stage = ld_stage == STAGES - 1 ? 0 : ld_stage + 1;
    find_tile();
  };
  if (lane == 0) met_bad_page[warp] = 0;
  ld_live = true;
  ld_t = ld.t1;  // none yet
  find_tile();

  uint4 qraw[kQv];
  // q of a segment as it lies; rows behind the last are zero and never written out
  auto load_q = [&](const Segment& n) {
#pragma unroll
    for (int k = 0; k < kQv; ++k) {
      const int v = threadIdx.x + k * kThreads;
      const int r = v / kVec, x = v % kVec, row = n.row0 + r;
      qraw[k] = make_uint4(0u, 0u, 0u, 0u);
      if (r < ROWS && row < n.rows_valid) {
        const int i = row / p.group, h = n.kvh * p.group + row - i * p.group;
        const long long at = n.b * p.q_sb + i * p.q_st + h * p.q_sh + x * 8;
        qraw[k] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + at));
      }
    }
  };
  Segment n;
  bool more = walk.next(p, prefix, n);
  if (!more) return;  // a range within a unit's empty places
  load_q(n);
#pragma unroll
  for (int x = 0; x < STAGES; ++x) load_tile();
  int stage = 0;

  for (bool first = true; more; first = false) {
    const Segment cur = n;
    const Seq s = cur.s;
    const int row0 = cur.row0, rows_valid = cur.rows_valid, t1 = cur.t1;

    // q rows into shared memory as halves times a power of two, in the order the products take the head dimension:
    // position 64 j + 16 cq + e holds dim 128 (j / 2) + 32 cq + 16 (j % 2) + e (D = 64: unchanged)
#pragma unroll
    for (int k = 0; k < kQv; ++k) {
      const int v = threadIdx.x + k * kThreads;
      const int r = v / kVec, x = v % kVec;
      if ((k + 1) * kThreads > ROWS * kVec && r >= ROWS) break;  // whole warps
      const uint32_t ws[4] = {qraw[k].x, qraw[k].y, qraw[k].z, qraw[k].w};
      float f[8], amax = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 w = p.bf16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&ws[e]))
                                : __half22float2(*reinterpret_cast<const __half2*>(&ws[e]));
        f[2 * e] = w.x;
        f[2 * e + 1] = w.y;
        amax = fmaxf(amax, fmaxf(fabsf(w.x), fabsf(w.y)));
      }
#pragma unroll
      for (int o = kVec / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const int e2 = max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -100);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e2) << 23);
      if (x == 0) row_factor[r] = __uint_as_float(static_cast<uint32_t>(127 - 14 + e2) << 23) * p.scale_log2;
      uint4 hq;
      hq.x = half2_bits(f[0] * up, f[1] * up);
      hq.y = half2_bits(f[2] * up, f[3] * up);
      hq.z = half2_bits(f[4] * up, f[5] * up);
      hq.w = half2_bits(f[6] * up, f[7] * up);
      const int at = D == 64 ? x * 8 : 64 * (2 * (x >> 4) + ((x >> 1) & 1)) + 16 * ((x >> 2) & 3) + 8 * (x & 1);
      *reinterpret_cast<uint4*>(qs + r * S::kQStride + at) = hq;
    }
    __syncthreads();

    // this lane's rows (columns of the products): 8 nt + 2 cq + {0, 1}
    // m is the largest score s_j so far, the sum's reference; mv the largest s_j + log2 vs_j, the accumulators': a block counts by
    // its softmax weight times its scale, so one of little weight cannot take the others' bits (kept within m - kSpan and
    // m + kRise: the factor between the two is a normal number)
    float factor[NT][2], m[NT][2], mv[NT][2], l[NT][2];
    int lim[NT][2];
    int min_lim = s.end;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = nt * 8 + 2 * cq + e;
        factor[nt][e] = row_factor[r];
        lim[nt][e] = row0 + r < rows_valid ? s.start + (row0 + r) / p.group + 1 : s.end;
        min_lim = min(min_lim, lim[nt][e]);
        m[nt][e] = mv[nt][e] = -INFINITY;
        l[nt][e] = 0.0f;
      }
    }
    min_lim = __reduce_min_sync(0xffffffffu, min_lim);
    float acc[NT][D / 16][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < D / 16; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][x][e] = 0.0f;

    int t = cur.t0 + warp;
    const bool any = t < t1;
    for (; t < t1; t += W) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      __syncwarp();
      const uint8_t* kt = ring + stage * S::kStageBytes;
      const uint8_t* vt = kt + TOK * D;
      float ks[MT], vs[MT], lv[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        ks[mt] = scales[stage * 2 * MT + mt];
        vs[mt] = scales[stage * 2 * MT + MT + mt];
        lv[mt] = lg2_abs(vs[mt]);
      }
      // scores: two accumulators per product shorten the dependent chain
      float sc[MT][NT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 8; ++e) sc[mt][nt][e >> 2][e & 3] = 0.0f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        uint32_t qf[NT][8];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint4* src = reinterpret_cast<const uint4*>(qs + (nt * 8 + g) * S::kQStride + 64 * j + 16 * cq);
          const uint4 a = src[0], d = src[1];
          qf[nt][0] = a.x; qf[nt][1] = a.y; qf[nt][2] = a.z; qf[nt][3] = a.w;
          qf[nt][4] = d.x; qf[nt][5] = d.y; qf[nt][6] = d.z; qf[nt][7] = d.w;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const uint8_t* kp = kt + mt * 16 * D + (j >> 1) * 128 + k_off[j & 1];
          const uint4 lo = *reinterpret_cast<const uint4*>(kp);
          const uint4 hi = *reinterpret_cast<const uint4*>(kp + 8 * D);
          const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t a0, a1, a2, a3;
            widen4<E4M3>(wl[x], a0, a2);
            widen4<E4M3>(wh[x], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(sc[mt][nt][x & 1], a0, a1, a2, a3, qf[nt][2 * x], qf[nt][2 * x + 1]);
          }
        }
      }
      // softmax: a lane has tokens g and g + 8 of each subtile for its rows
      float top[NT][2], topv[NT][2];
      const bool tail = t * TOK + TOK > min_lim;  // some token is hidden from some row
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sc[mt][nt][0][e] = (sc[mt][nt][0][e] + sc[mt][nt][1][e]) * (ks[mt] * factor[nt][e & 1]);
      if (tail) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (t * TOK + mt * 16 + (e >> 1) * 8 + g >= lim[nt][e & 1]) sc[mt][nt][0][e] = -INFINITY;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[nt][e] = fmaxf(sc[0][nt][0][e], sc[0][nt][0][2 + e]);
          topv[nt][e] = top[nt][e] + lv[0];
#pragma unroll
          for (int mt = 1; mt < MT; ++mt) {
            const float a = fmaxf(sc[mt][nt][0][e], sc[mt][nt][0][2 + e]);
            top[nt][e] = fmaxf(top[nt][e], a);
            topv[nt][e] = fmaxf(topv[nt][e], a + lv[mt]);
          }
        }
      }
      bool grew = false;
      float ref[NT][2], down[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) top[nt][e] = fmaxf(top[nt][e], __shfl_xor_sync(0xffffffffu, top[nt][e], o));
          if constexpr (MT == 1) {
            topv[nt][e] = top[nt][e] + lv[0];
          } else {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) topv[nt][e] = fmaxf(topv[nt][e], __shfl_xor_sync(0xffffffffu, topv[nt][e], o));
          }
          top[nt][e] = fmaxf(top[nt][e], m[nt][e]);
          topv[nt][e] = fminf(fmaxf(fmaxf(topv[nt][e], mv[nt][e]), top[nt][e] - kSpan), top[nt][e] + kRise);
          grew |= top[nt][e] > m[nt][e] || topv[nt][e] > mv[nt][e];
          ref[nt][e] = top[nt][e] == -INFINITY ? 0.0f : top[nt][e];  // a row that has seen nothing yet
          down[nt][e] = ex2(ref[nt][e] - (topv[nt][e] == -INFINITY ? 0.0f : topv[nt][e]));
        }
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          l[nt][0] *= ex2(m[nt][0] - ref[nt][0]);
          l[nt][1] *= ex2(m[nt][1] - ref[nt][1]);
          m[nt][0] = top[nt][0];
          m[nt][1] = top[nt][1];
          const float a0 = topv[nt][0] == -INFINITY ? 0.0f : ex2(mv[nt][0] - topv[nt][0]);
          const float a1 = topv[nt][1] == -INFINITY ? 0.0f : ex2(mv[nt][1] - topv[nt][1]);
          mv[nt][0] = topv[nt][0];
          mv[nt][1] = topv[nt][1];
#pragma unroll
          for (int x = 0; x < D / 16; ++x) {
            acc[nt][x][0] *= a0;
            acc[nt][x][1] *= a1;
            acc[nt][x][2] *= a0;
            acc[nt][x][3] *= a1;
          }
        }
      }
      uint32_t pb[MT][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float off[2] = {ref[nt][0] - kShift, ref[nt][1] - kShift};
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sc[mt][nt][0][e] = ex2(sc[mt][nt][0][e] - off[e & 1]);
            l[nt][e & 1] += sc[mt][nt][0][e];
          }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // (in this order: a weight is at most 2^14, so times 2^kSpan finite)
            float w0 = sc[mt][nt][0][half * 2] * down[nt][0] * vs[mt], w1 = sc[mt][nt][0][half * 2 + 1] * down[nt][1] * vs[mt];
            if (tail) {  // a hidden token weighs nothing even where its block's scale is NaN
              const int tok = t * TOK + mt * 16 + half * 8 + g;
              w0 = tok >= lim[nt][0] ? 0.0f : w0;
              w1 = tok >= lim[nt][1] ? 0.0f : w1;
            }
            pb[mt][nt][half] = transpose8x8(half2_bits(w0, w1));
          }
        }
      }
      // Tokens that some rows see and others do not: 0 * NaN would stay in the others' products, so a NaN byte among their values
      // becomes zero here and NaN in that dimension of the rows that see it.  (Tokens that all rows see need no such care.)
      if constexpr (E4M3) {
        if (tail && min_lim < s.end) {
          uint8_t* vw = ring + stage * S::kStageBytes + TOK * D;
          const int lo = max(min_lim - t * TOK, 0), hi = min(s.end - t * TOK, TOK);
          bool found = false;
          for (int v = lane; v < (hi - lo) * (D / 16); v += 32) {
            const uint4 w = *reinterpret_cast<const uint4*>(vw + tile_chunk<D>(lo + v / (D / 16), v % (D / 16)));
            found |= (nan_bytes(w.x) | nan_bytes(w.y) | nan_bytes(w.z) | nan_bytes(w.w)) != 0;
          }
          if (__any_sync(0xffffffffu, found)) {
            constexpr int X = D == 64 ? 2 : 4;  // words of this lane's dims, as in the products below
            for (int r = lo; r < hi; ++r) {
#pragma unroll
              for (int jj = 0; jj < (D + 127) / 128; ++jj) {
                uint32_t* src = reinterpret_cast<uint32_t*>(
                    vw + (D == 64 ? tile_chunk<D>(r, g >> 1) + (g & 1) * 8 : tile_chunk<D>(r, 8 * jj + g)));
                uint32_t nan[X];
#pragma unroll
                for (int x = 0; x < X; ++x) {
                  nan[x] = nan_bytes(src[x]);
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int y = 0; y < 4; ++y)
#pragma unroll
                      for (int e = 0; e < 2; ++e)
                        if ((nan[x] >> (8 * y + 7) & 1) != 0 && t * TOK + r < lim[nt][e]) acc[nt][2 * (4 * jj + x) + (y >> 1)][2 * (y & 1) + e] = nan_f();
                }
                __syncwarp();
                if (cq == 0) {
#pragma unroll
                  for (int x = 0; x < X; ++x) src[x] &= ~((nan[x] >> 7) * 0xffu);
                }
              }
            }
            __syncwarp();
          }
        }
      }
      // o^T += v^T p^T: a lane has tokens 2 cq + {0, 1, 8, 9} of each subtile and D / 8 dims
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const uint8_t* vm = vt + mt * 16 * D;
#pragma unroll
        for (int jj = 0; jj < (D + 127) / 128; ++jj) {
          constexpr int X = D == 64 ? 2 : 4;  // words of four dims
          uint32_t w[4][X];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint8_t* vp = vm + (i >> 1) * 8 * D + v_off[i & 1];  // token 2 cq + {0, 1, 8, 9}[i]
            if constexpr (D == 64) {
              const uint2 v = *reinterpret_cast<const uint2*>(vp);
              w[i][0] = v.x;
              w[i][1] = v.y;
            } else {
              const uint4 v = *reinterpret_cast<const uint4*>(vp + 128 * jj);
              w[i][0] = v.x;
              w[i][1] = v.y;
              w[i][2] = v.z;
              w[i][3] = v.w;
            }
          }
#pragma unroll
          for (int x = 0; x < X; ++x) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {  // dims 4x + 2y, 4x + 2y + 1
              uint32_t a0, a1, a2, a3;
              widen4<E4M3>(__byte_perm(w[0][x], w[1][x], y == 0 ? 0x5140 : 0x7362), a0, a1);
              widen4<E4M3>(__byte_perm(w[2][x], w[3][x], y == 0 ? 0x5140 : 0x7362), a2, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816(acc[nt][2 * (4 * jj + x) + y], a0, a1, a2, a3, pb[mt][nt][0], pb[mt][nt][1]);
            }
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      if (t + W < t1) {
        load_tile();
        stage = stage == STAGES - 1 ? 0 : stage + 1;
      }
    }

    more = walk.next(p, prefix, n);
    if (more) load_q(n);  // on its way while this segment's warps are joined
    // join the warps: 8 rows at a time through the stage each has just used up, which is loaded again afterwards
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float* dst = reinterpret_cast<float*>(ring + stage * S::kStageBytes);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], o);
        const int r = 2 * cq + e;
        if (g == 0) {
          warp_m[warp][nt * 8 + r] = m[nt][e];
          warp_l[warp][nt * 8 + r] = l[nt][e];
          warp_mv[warp][nt * 8 + r] = mv[nt][e];
        }
        if (any) {
          // dims of acc[2x], acc[2x + 1]: D 64: 8 g + 4 x; else 128 (x / 4) + 16 g + 4 (x % 4), four in a row
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {
            const int chunk = D == 64 ? 2 * g + x : 32 * (x / 4) + 4 * g + x % 4;
            *reinterpret_cast<float4*>(dst + r * D + 4 * merge_chunk<D>(r, chunk)) =
                make_float4(acc[nt][2 * x][e], acc[nt][2 * x][2 + e], acc[nt][2 * x + 1][e], acc[nt][2 * x + 1][2 + e]);
          }
        }
      }
      if (lane == 0) warp_at[warp] = static_cast<int>(reinterpret_cast<uint8_t*>(dst) - smem);
      __syncthreads();
      const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (first ? 0 : 1);
      const int nw = min(W, t1 - cur.t0);  // warps that had a tile
      if (threadIdx.x < 128) {  // a row's maximum and sum, 16 lanes each; warp_m becomes what a warp's rows are multiplied by
        const int r = nt * 8 + (threadIdx.x >> 4), i = threadIdx.x & 15;
        const float mi = i < nw ? warp_m[i][r] : -INFINITY, mvi = i < nw ? warp_mv[i][r] : -INFINITY;
        float top = mi, topv = mvi;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          topv = fmaxf(topv, __shfl_xor_sync(0xffffffffu, topv, o));
        }
        const float w = ex2(mi - (top == -INFINITY ? 0.0f : top));
        float sum = i < nw ? w * warp_l[i][r] : 0.0f;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float refv = topv == -INFINITY ? 0.0f : topv;
        if (i < nw) warp_m[i][r] = ex2(mvi - refv) * (sum == 0.0f ? 0.0f : 1.0f / sum);
        if (i == 0) {
          row_top[r] = top;
          row_sum[r] = sum;
          // what is left of the accumulators' reference, 2^(refv - top), in two halves: subnormal outputs keep their bits
          row_up[r] = ex2(0.5f * (refv - (top == -INFINITY ? refv : top)));
        }
      }
      __syncthreads();
      constexpr int kOut = 8 * (D / 4);
#pragma unroll
      for (int k = 0; k < (kOut + kThreads - 1) / kThreads; ++k) {
        const int v = threadIdx.x + k * kThreads;
        const int r8 = v / (D / 4), x = v % (D / 4);
        const int r = nt * 8 + r8, row = row0 + r;
        if (v >= kOut || row >= rows_valid) break;
        float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int i = 0; i < nw; ++i) {
          const float4 a = *reinterpret_cast<const float4*>(smem + warp_at[i] + r8 * D * 4 + 16 * merge_chunk<D>(r8, x));
          const float w = warp_m[i][r];
          o[0] += a.x * w;
          o[1] += a.y * w;
          o[2] += a.z * w;
          o[3] += a.w * w;
        }
        const float top = row_top[r], sum = row_sum[r], up = row_up[r];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = o[e] * up * up;
        if (cur.whole) {
          const int i = row / p.group, h = cur.kvh * p.group + row - i * p.group;
          const size_t orow = (static_cast<size_t>(cur.b) * p.tokens + i) * p.hq + h;
          store_out4(p, orow * D + 4 * x, o);
          if (p.lse != nullptr && x == 0) p.lse[orow] = lse_of(top == -INFINITY ? 0.0f : top, sum);
        } else {
          *reinterpret_cast<float4*>(p.part_o + (slot * ROWS + r) * D + 4 * x) = make_float4(o[0], o[1], o[2], o[3]);
          if (x == 0) p.part_ml[slot * ROWS + r] = make_float2(top, sum);
        }
      }
      __syncthreads();
    }
    if (any) {
      load_tile();
      stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (lane == 0 && met_bad_page[warp] != 0) report_bad(p.status);
}

// ------------------------------------------------------------------------------------ joining cut units
// Rows of units that range borders cut (partials of CTAs c0 .. c1), rows that see nothing (zeros) and rows of
// sequences whose lengths do not fit (NaN).  A CTA takes up to 8 rows, a warp each; a row with many partials is
// joined by the whole CTA, and where there are few rows by gridDim.y CTAs, each a share of the columns.
template <int D, int NT>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const AttnParams p, int rows_per_cta) {
  using S = Shape<D, NT>;
  constexpr int TOK = S::kTok, ROWS = S::kRows, kShort = 8;
  constexpr int TPR = D / 4;               // threads of a row
  const int tpr = TPR / gridDim.y;         // threads of this CTA's share of a row
  const int pg_n = kJoinThreads / tpr;     // partials at a time
  extern __shared__ __align__(128) uint8_t smem[];
  float* weight = reinterpret_cast<float*>(smem);                       // [kMaxCtas]
  float4* sums = reinterpret_cast<float4*>(smem + kMaxCtas * 4);        // [pg_n][tpr]
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem + kMaxCtas * 4 + kJoinThreads * 16);
  __shared__ uint32_t scratch[kJoinThreads / 32];
  __shared__ float red[2][kJoinThreads / 32];
  __shared__ uint32_t long_c0[8], long_c1[8], long_t0[8];
  __shared__ int long_r[8];
  __shared__ int long_row[8];

  make_plan<TOK, ROWS, kJoinThreads>(p, prefix, scratch);
  const uint32_t total = prefix[p.c.batch];
  const uint32_t ctas = active_ctas(p, total);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = p.c.batch * p.tokens * p.hq;
  const int step = gridDim.x * rows_per_cta;
  bool waited = false;  // the rows are found from the call's inputs alone, while the attention kernel still runs
  auto wait_partials = [&]() {
    if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
    waited = true;
  };
  for (int base = blockIdx.x * rows_per_cta; base < rows; base += step) {
    const int row = base + warp;
    if (lane == 0) long_c1[warp] = 0;
    if (warp < rows_per_cta && row < rows) {  // short rows: the first share's CTA does all of them
      const int rest = row / p.hq, h = row - rest * p.hq;
      const int i = rest % p.tokens, b = rest / p.tokens;
      const Seq s = load_seq(p.c, b, p.tokens);
      if (!s.ok || i >= s.end - s.start) {
        const float f = s.ok ? 0.0f : nan_f();
        const float o[4] = {f, f, f, f};
        for (int x = lane; x < TPR && blockIdx.y == 0; x += 32) store_out4(p, static_cast<size_t>(row) * D + 4 * x, o);
        if (p.lse != nullptr && lane == 0 && blockIdx.y == 0) p.lse[row] = s.ok ? -INFINITY : nan_f();
      } else {
        const Unit u = unit_of<TOK, ROWS>(p, s);
        const int kvh = h / p.group, r = i * p.group + h - kvh * p.group;
        const uint32_t first = prefix[b] + static_cast<uint32_t>(kvh * u.row_tiles + r / ROWS) * u.length;
        const uint32_t c0 = cta_of(first + kUnitCost<TOK>, total, ctas), c1 = cta_of(first + u.length - 1, total, ctas);
        const int rr = r % ROWS;
        if (c1 - c0 >= kShort) {
          if (lane == 0) {
            long_c0[warp] = c0;
            long_c1[warp] = c1;
            long_t0[warp] = first;
            long_r[warp] = rr;
            long_row[warp] = row;
          }
        } else if (c1 > c0 && blockIdx.y == 0) {
          // the partial of a CTA is its first segment's, unless the unit began inside the CTA's range
          const uint32_t slot0 = 2 * c0 + (range_begin(c0, total, ctas) >= first ? 0 : 1);
          const size_t slot = lane == 0 ? slot0 : 2 * (c0 + min(static_cast<uint32_t>(lane), c1 - c0));
          wait_partials();
          const int n = static_cast<int>(c1 - c0) + 1;
          const float2 ml = lane < n ? __ldcg(&p.part_ml[slot * ROWS + rr]) : make_float2(-INFINITY, 0.0f);
          constexpr int X = (TPR + 31) / 32;
          float4 part[kShort][X];
#pragma unroll
          for (int k = 0; k < kShort; ++k) {
            const size_t sk = k == 0 ? slot0 : 2 * (c0 + k);
            const float4* src = reinterpret_cast<const float4*>(p.part_o + (sk * ROWS + rr) * D);
#pragma unroll
            for (int x = 0; x < X; ++x)
              part[k][x] = k < n && lane + 32 * x < TPR ? __ldcg(src + lane + 32 * x) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          }
          float top = ml.x;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const float ref = top == -INFINITY ? 0.0f : top;
          const float w = ex2(ml.x - ref) * ml.y;
          float sum = w;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          float acc[X][4];
#pragma unroll
          for (int x = 0; x < X; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[x][e] = 0.0f;
#pragma unroll
          for (int k = 0; k < kShort; ++k) {
            const float wk = __shfl_sync(0xffffffffu, w, k) * inv;
            if (k < n) {
#pragma unroll
              for (int x = 0; x < X; ++x) {
                acc[x][0] += wk * part[k][x].x;
                acc[x][1] += wk * part[k][x].y;
                acc[x][2] += wk * part[k][x].z;
                acc[x][3] += wk * part[k][x].w;
              }
            }
          }
#pragma unroll
          for (int x = 0; x < X; ++x)
            if (lane + 32 * x < TPR) store_out4(p, static_cast<size_t>(row) * D + 4 * (lane + 32 * x), acc[x]);
          if (p.lse != nullptr && lane == 0) p.lse[row] = lse_of(ref, sum);
        }
      }
    }
    __syncthreads();
    for (int k = 0; k < rows_per_cta; ++k) {  // uniform over the CTA
      const uint32_t c0 = long_c0[k], c1 = long_c1[k];
      if (c1 == 0) continue;
      wait_partials();
      const int n = static_cast<int>(c1 - c0) + 1, rr = long_r[k];
      const uint32_t first = long_t0[k];
      // only the first CTA's partial may lie in its second slot
      const size_t slot0 = 2 * static_cast<size_t>(c0) + (range_begin(c0, total, ctas) >= first ? 0 : 1);
      auto slot_of = [&](int x) { return x == 0 ? slot0 : 2 * static_cast<size_t>(c0 + x); };
      const int x = threadIdx.x % tpr, pg = threadIdx.x / tpr;
      const int col = (blockIdx.y * tpr + x) * 4;
      auto load_part = [&](int y) {
        return __ldcg(reinterpret_cast<const float4*>(p.part_o + (slot_of(y) * ROWS + rr) * D + col));
      };
      constexpr int kEarly = 8;  // partials on their way while the weights are formed
      float4 early[kEarly];
#pragma unroll
      for (int i = 0; i < kEarly; ++i)
        early[i] = pg + i * pg_n < n ? load_part(pg + i * pg_n) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      constexpr int M = (kMaxCtas + kJoinThreads - 1) / kJoinThreads;
      float2 ml[M];
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < M; ++i) {
        const int y = threadIdx.x + i * kJoinThreads;
        ml[i] = y < n ? __ldcg(&p.part_ml[slot_of(y) * ROWS + rr]) : make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, ml[i].x);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (lane == 0) red[0][warp] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kJoinThreads / 32; ++w) top = fmaxf(top, red[0][w]);
      const float ref = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < M; ++i) {
        const int y = threadIdx.x + i * kJoinThreads;
        const float w = ex2(ml[i].x - ref) * ml[i].y;
        if (y < n) weight[y] = w;
        sum += w;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) red[1][warp] = sum;
      __syncthreads();
      sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kJoinThreads / 32; ++w) sum += red[1][w];
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      auto add = [&](float w, const float4& v) {
        a.x += w * v.x;
        a.y += w * v.y;
        a.z += w * v.z;
        a.w += w * v.w;
      };
#pragma unroll
      for (int i = 0; i < kEarly; ++i)
        if (pg + i * pg_n < n) add(weight[pg + i * pg_n] * inv, early[i]);
#pragma unroll 4
      for (int y = pg + kEarly * pg_n; y < n; y += pg_n) add(weight[y] * inv, load_part(y));
      sums[pg * tpr + x] = a;
      __syncthreads();
      if (pg == 0) {
        float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int y = 0; y < pg_n; ++y) {
          const float4 v = sums[y * tpr + x];
          o[0] += v.x;
          o[1] += v.y;
          o[2] += v.z;
          o[3] += v.w;
        }
        store_out4(p, static_cast<size_t>(long_row[k]) * D + col, o);
        if (p.lse != nullptr && col == 0) p.lse[long_row[k]] = lse_of(ref, sum);
      }
      __syncthreads();  // before the next row's weights and sums
    }
    __syncthreads();  // before the next rows' descriptions
  }
  wait_partials();
}

constexpr int kSmallWarps = 4;  // warps of a CTA where there are many units

template <int D, int NT>
struct Tag {
  static constexpr int kD = D, kNt = NT;
};

template <int D, int NT>
size_t workspace_bytes(int sms) {
  using S = Shape<D, NT>;
  const size_t slots = 2 * static_cast<size_t>(sms) * (S::kWarpsPerSm / kSmallWarps);
  return slots * S::kRows * (D * 4 + 8);
}

template <int D, bool E4M3, int NT, int W>
int launch_with(const char* who, AttnParams& p, int sms, int single_units, void* workspace, cudaStream_t s) {
  using S = Shape<D, NT>;
  p.single = single_units > 0;
  p.grid = p.single ? single_units : sms * (S::kWarpsPerSm / W);
  p.min_tiles = W == kSmallWarps ? kSmallWarps : 8;
  if (!p.single && p.grid > kMaxCtas) return fail(TOKMIX_ERR_UNSUPPORTED, "%s: more SMs than the kernel is planned for", who);
  const size_t slots = 2 * static_cast<size_t>(p.grid);
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + slots * S::kRows * D);
  const int plan = p.single ? 0 : (p.c.batch + 1) * 4;
  const int join_smem = kMaxCtas * 4 + kJoinThreads * 16 + plan;
  const int plan_max = (kMaxBatch + 1) * 4;  // the limit is set once, for the largest batch
  const int attn_plan_max = W == kSmallWarps ? plan_max : (kMaxCtas + 1) * 4;  // large CTAs: at most a unit per SM
  auto* attn = attn_kernel<D, E4M3, NT, W>;
  auto* join = join_kernel<D, NT>;
  if (!ensure_smem_attr(reinterpret_cast<const void*>(attn), S::smem_bytes(W) + attn_plan_max) ||
      !ensure_smem_attr(reinterpret_cast<const void*>(join), kMaxCtas * 4 + kJoinThreads * 16 + plan_max))
    return fail(TOKMIX_ERR_LAUNCH, "%s: cannot set the shared memory size", who);
  p.row_lines = (p.c.max_pages + 31) / 32;
  p.table_lines = static_cast<int>(std::min<long long>(static_cast<long long>(p.row_lines) * p.c.batch, 32LL * W * p.grid));
  launch_overlapped(attn, dim3(p.grid), dim3(32 * W), S::smem_bytes(W) + plan, s, p);
  if (const int rc = check_launch(who)) return rc;
  if (p.single) return TOKMIX_OK;
  const long long rows = static_cast<long long>(p.c.batch) * p.tokens * p.hq;
  const int per = static_cast<int>(std::min<long long>(8, (rows + 2 * sms - 1) / (2 * sms)));
  const long long want = (rows + per - 1) / per;
  // few rows of long sequences are shared by CTAs of 64 columns; more CTAs than run at once would cost more (256 rows of 14
  // partials, D 256: 11.7 us, shared 18.8)
  const dim3 join_grid(static_cast<unsigned>(std::min<long long>(want, 4LL * sms)), rows * (D / 64) <= 2 * sms ? D / 64 : 1);
  launch_overlapped(join, join_grid, dim3(kJoinThreads), static_cast<size_t>(join_smem), s, p, per);
  return check_launch(who);
}

struct Layout {
  int single_units;  // a CTA per unit; 0: ranges of the line
  bool large;        // CTAs that have the SM to themselves
};

template <int D, int NT>
Layout layout_of(const AttnParams& p, int sms) {
  using S = Shape<D, NT>;
  const long long units = static_cast<long long>(p.c.batch) * p.c.hkv * ((p.tokens * p.group + S::kRows - 1) / S::kRows);
  // A CTA per unit, without a plan before it and a join behind it, where the table has room for short sequences only.  Up to
  // a unit per SM a unit's warps are all that read for it: 2 tiles a warp while most SMs have no unit, then 4, then 8 (planned
  // -> a CTA per unit; Hkv 8, D 128, 8 units of 1024 tokens, 3 tiles: 8.0 -> 9.3 us; 48 units, 3 tiles: 9.2 -> 9.3; 96 units:
  // 12.7 -> 10.7; D 256, 32 units of 1000 tokens, 6 tiles: 11.7 -> 14.4; D 128, 128 units of 2000, 6 tiles: 17.2 -> 16.2).
  // More units: a change of unit costs a range more than a CTA of its own, as long as no unit is long: up to 256 KB, or 512 KB
  // where there are enough units to even out the ends.  Ranges -> a CTA per unit, with lengths uniform up to the table's (u), a
  // tenth filling it and the others short (t), all filling it (f):
  //   D 128, 800 units,  256 KB:  u 32.0 -> 30.7 us, t 21.0 -> 20.5, f 44.0 -> 39.9
  //           240 units,  512 KB:  u 18.4 -> 27.0,    t 13.9 -> 23.2, f 30.3 -> 32.2
  //          1760 units,  512 KB:  u 88.1 -> 82.7,    t 51.9 -> 54.5, f 150 -> 142
  //   D 256, 160 units,  512 KB:  u 18.8 -> 21.7,    t 19.0 -> 22.3, f 23.3 -> 24.7
  //           400 units,  512 KB:  u 34.8 -> 30.2,    t 23.0 -> 26.4, f 49.3 -> 39.8
  const long long room = static_cast<long long>(p.c.max_pages) * p.c.page, most = (room + S::kTok - 1) / S::kTok;
  const int rounds = units * 4 <= sms ? 2 : units * 2 <= sms ? 4 : 8;
  if (units <= sms && most <= rounds * S::kWarpsPerSm) return {static_cast<int>(units), true};
  const long long slots = static_cast<long long>(sms) * (S::kWarpsPerSm / kSmallWarps);
  const long long bytes = (units * 4 >= (D == 256 ? 3 : 12) * slots ? 512 : 256) << 10;
  if (units > sms && units <= 1 << 20 && room * 2 * D <= bytes)  // (indexes of threads in 32 bits)
    return {static_cast<int>(units), false};
  // Few units: a CTA per SM leaves the fewest partial rows to join (8-row units, 1 unit of 64000 tokens, D 128: 14.8 to 14.8 us;
  // 2: 16.6 to 18.5; 4: 20.3 to 21.3; 16-row units, D 256, 8: 37 to 39; 32: 48 to 53).  Many: small CTAs, whose changes of unit
  // overlap (8-row units, D 64, 8: 13.3 to 14.6 us; D 128, 32: 28.5 to 30.3; 16-row units, D 128, 64: 30.3 to 31.4).
  return {0, units * (NT == 1 ? 32 : 4) <= sms};
}

template <int D, bool E4M3, int NT>
int launch_attn(const char* who, AttnParams& p, int sms, void* workspace, cudaStream_t s) {
  const Layout l = layout_of<D, NT>(p, sms);
  return l.large ? launch_with<D, E4M3, NT, Shape<D, NT>::kWarpsPerSm>(who, p, sms, l.single_units, workspace, s)
                 : launch_with<D, E4M3, NT, kSmallWarps>(who, p, sms, l.single_units, workspace, s);
}

template <int D>
int dispatch_attn(const char* who, AttnParams& p, bool e4m3, int sms, void* ws, cudaStream_t s) {
  // up to 8 query rows share a pass (8 columns of the product), else 16
  if (p.tokens * p.group <= 8)
    return e4m3 ? launch_attn<D, true, 1>(who, p, sms, ws, s) : launch_attn<D, false, 1>(who, p, sms, ws, s);
  return e4m3 ? launch_attn<D, true, 2>(who, p, sms, ws, s) : launch_attn<D, false, 2>(who, p, sms, ws, s);
}

// f(Tag<D, NT>) of a call's shape: up to 8 query rows share a pass (8 columns of the product), else 16
template <typename F>
long long of_shape(int head_dim, long long rows_per_head, F f) {
  const bool one = rows_per_head <= 8;
  if (head_dim == 64) return one ? f(Tag<64, 1>{}) : f(Tag<64, 2>{});
  if (head_dim == 128) return one ? f(Tag<128, 1>{}) : f(Tag<128, 2>{});
  return one ? f(Tag<256, 1>{}) : f(Tag<256, 2>{});
}

// Bytes of workspace that a call needs: none where each unit has a CTA of its own
long long workspace_of(const AttnParams& p, int head_dim, int sms) {
  return of_shape(head_dim, static_cast<long long>(p.tokens) * p.group, [&](auto t) -> long long {
    constexpr int D = decltype(t)::kD, NT = decltype(t)::kNt;
    return layout_of<D, NT>(p, sms).single_units > 0 ? 0 : workspace_bytes<D, NT>(sms);
  });
}

}  // namespace kv8
}  // namespace tokmix

extern "C" long long tokmix_kv8_attention_workspace_bytes(int tokens, int heads_q, int heads_kv, int head_dim) {
  using namespace tokmix;
  using namespace tokmix::kv8;
  if (tokens < 1 || tokens > kMaxTokens || heads_kv <= 0 || heads_q <= 0 || heads_q % heads_kv != 0 ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return -1;
  const int sms = device_sm_count();
  return of_shape(head_dim, static_cast<long long>(tokens) * (heads_q / heads_kv), [&](auto t) -> long long {
    return workspace_bytes<decltype(t)::kD, decltype(t)::kNt>(sms);
  });
}

extern "C" long long tokmix_kv8_attention_workspace_bytes_for(int tokens, int heads_q, int heads_kv, int head_dim, int batch,
                                                              int max_pages, int page_size) {
  using namespace tokmix;
  using namespace tokmix::kv8;
  const long long most = tokmix_kv8_attention_workspace_bytes(tokens, heads_q, heads_kv, head_dim);
  if (most < 0 || batch < 0 || max_pages < 0 || page_size <= 0) return -1;
  if (batch == 0) return 0;
  if (batch > kMaxBatch || heads_q > 65536) return most;  // the call itself refuses them
  AttnParams p{};
  p.tokens = tokens;
  p.group = heads_q / heads_kv;
  p.c.batch = batch;
  p.c.hkv = heads_kv;
  p.c.max_pages = max_pages;
  p.c.page = page_size;
  return workspace_of(p, head_dim, device_sm_count());
}

extern "C" int tokmix_kv8_attention(const void* q, long long q_batch_stride, long long q_token_stride,
                                    long long q_head_stride, void* out, float* lse, int tokens, int heads_q,
                                    int io_dtype, float sm_scale, const tokmix_kv8_cache* cache, void* workspace,
                                    long long workspace_bytes, uint32_t* status, void* stream) {
  using namespace tokmix;
  using namespace tokmix::kv8;
  const char* who = "tokmix_kv8_attention";
  AttnParams p{};
  if (const int rc = make_view(who, cache, p.c)) return rc;
  if (tokens < 0 || tokens > kMaxTokens)
    return fail(TOKMIX_ERR_UNSUPPORTED, "%s: at most %d new tokens per sequence (got %d)", who, kMaxTokens, tokens);
  if (heads_q <= 0 || heads_q % cache->heads_kv != 0)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: heads_q (%d) must be a multiple of heads_kv (%d)", who, heads_q,
                cache->heads_kv);
  if (io_dtype != TOKMIX_DTYPE_BF16 && io_dtype != TOKMIX_DTYPE_FP16)
    return fail(TOKMIX_ERR_UNSUPPORTED, "%s: q is bf16 or fp16 (dtype %d)", who, io_dtype);
  if (!(sm_scale > 0.0f) || !std::isfinite(sm_scale))
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: sm_scale must be positive and finite", who);
  if (tokens == 0 || p.c.batch == 0) return TOKMIX_OK;
  if (!q || !out) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: null pointer argument", who);
  if (reinterpret_cast<uintptr_t>(q) % 16 != 0 || reinterpret_cast<uintptr_t>(out) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: tensors must be 16-byte aligned", who);
  for (const long long st : {q_batch_stride, q_token_stride, q_head_stride})
    if (st % 8 != 0 || st < 0)
      return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: strides of q must be multiples of 8 elements", who);
  if (p.c.batch > kMaxBatch) return fail(TOKMIX_ERR_UNSUPPORTED, "%s: at most %d sequences (got %d)", who, kMaxBatch, p.c.batch);
  const long long most_tiles = ((static_cast<long long>(p.c.max_pages) * p.c.page + 15) / 16 + kUnitCost<32>) * p.c.hkv *
                               ((static_cast<long long>(tokens) * (heads_q / p.c.hkv) + 7) / 8) * p.c.batch;
  if (heads_q > 65536 || most_tiles > 0x7fffffffLL || static_cast<long long>(p.c.batch) * tokens * heads_q > 0x3fffffffLL)
    return fail(TOKMIX_ERR_UNSUPPORTED, "%s: problem too large", who);
  if (const int rc = check_device()) return rc;
  p.q = q;
  p.q_sb = q_batch_stride;
  p.q_st = q_token_stride;
  p.q_sh = q_head_stride;
  p.out = out;
  p.lse = lse;
  p.tokens = tokens;
  p.hq = heads_q;
  p.group = heads_q / cache->heads_kv;
  p.bf16 = io_dtype == TOKMIX_DTYPE_BF16;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool e4m3 = cache->dtype == TOKMIX_DTYPE_E4M3;
  const int sms = device_sm_count();
  const long long need = workspace_of(p, cache->head_dim, sms);
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: workspace of %lld bytes, %lld needed", who, workspace ? workspace_bytes : 0, need);
  if (cache->head_dim == 64) return dispatch_attn<64>(who, p, e4m3, sms, workspace, s);
  if (cache->head_dim == 128) return dispatch_attn<128>(who, p, e4m3, sms, workspace, s);
  return dispatch_attn<256>(who, p, e4m3, sms, workspace, s);
}
