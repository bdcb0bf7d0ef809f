// fa2_bwd.cu -- gradient of the attention forward (fa2_fwd.cu) for sm_100a (B200).
//
// With c = sm_scale and the forward's lse (natural logarithm), for every query head:
//   P = exp(c q k^T - lse) under the mask,  delta = sum_d do * o  (a row each)
//   dv = P^T do,   dS = P * (do v^T - delta),   dq = c dS k,   dk = c dS^T q
// dk and dv are summed over the query heads that share a key/value head.  P is formed again from
// q, k and lse, so the forward keeps one number per row instead of the S x S matrix.
//
// Three launches:
//   fa2_bwd_prep    -delta and -lse * log2(e) in rows padded to whole query tiles (padding: 0, -inf,
//                   so that a padded row's P is 0), the counters below set to 0.
//   fa2_bwd_kernel  persistent, one CTA per SM.  A unit is a tile of 128 keys of one key/value head: K and V
//                   stay in shared memory, the tiles of kBQ queries of every query head of the group
//                   pass by (last tile first), and dK and dV grow in TMEM.  Scores are held
//                   transposed, keys along the 128 TMEM lanes:
//     S^T  = K Q^T     (SS)            P^T = 2^(c log2e S^T - lse2), bf16, over S^T's own columns
//     dV  += P^T dO    (A from TMEM)
//     dP^T = V dO^T    (SS)            dS^T = P^T * (dP^T - delta), bf16, into shared memory
//     dK  += dS^T Q    (SS)
//     dQ   = dS K      (SS; A is the same dS^T tile read MN-major)
//   A query tile's dQ is the sum over key tiles, that is, over CTAs.  It grows in fp32 in global
//   memory by vector reductions, in the order of the key tiles: a CTA waits until the query tile's
//   turn counter names its key tile, adds, and passes the turn on.  So the bits are the same every
//   time; the first tile stores instead of adding (no clearing pass).
//   Units are taken from a counter in an order in which a unit waits only for units taken earlier, by
//   CTAs that are running, so the waits end with any number of resident CTAs.
//   fa2_bwd_finish  dq = c times those sums, rounded, in dq's layout, and dV and dK of key tiles that came
//                   in parts.  (The last key tile's CTA could finish dq in passing, but reading the sums back held its pipeline
//                   up for 10 000 to 20 000 cycles a tile.  With a single key tile dQ is written at once.)
// Roles: two softmax warpgroups (four at D 64), each a share of a tile's query columns (TMEM is read in the layout of mma
// accumulators, in which a lane has two of every 8 columns: a lane that owned a row read every row statistic as a broadcast,
// 1400 of a step's cycles of shared memory); four dQ warps (TMEM to global); a warp each for TMA and the unit counter, for the
// MMAs and TMEM, for passing on and for awaiting the turns of the dQ sums.
// Order of the MMAs:  dP(t) dV(t) S(t+1) dQ(t) dK(t) | dP(t+1) ...: while the softmax warps form P
// the tensor core has dQ and dK to do, and while they form dS it has dV and the next S.  At D 64, where dQ has columns of
// its own, dP(t+1) goes before dQ(t).
//
// What bounds it (D 128, a step of 128 queries x 128 keys, cycles): the tensor core 2560, shared memory about 3200, sending
// 64 KB of dQ 2600 at the 25 bytes a cycle that an SM sends; measured 4300 to 4600, and under sustained load the
// clock, which falls at 1000 W.  B4 Hq32 Hkv8 S8192 causal 6.2 to 6.3 ms, 870 to 890 TFLOP/s of 1384 sustained; without dQ's way to
// memory it took 5.0 ms.
//
// head_dim 256: dV and dK of 128 keys alone would fill TMEM (2 x 256 columns), so a unit takes half
// of their columns (and of dQ's) and forms S and dP whole; queries come in tiles of 64.  V stays in
// TMEM as the A operand of dP (128 columns), which leaves shared memory room for two stages of Q and dO (32 KB
// each) beside K (64 KB), and takes V's rows out of what the tensor core reads there: at N = 64 an MMA
// with both operands in shared memory reads its full width, 128 bytes a cycle.  dQ is formed transposed
// (dQ^T = K^T dS^T), which keeps M at 128.
//
// Every wait is bounded (sm100.cuh): a stuck pipeline sets a status bit and the CTA drains.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "host_common.h"
#include "sm100.cuh"

namespace tokmix {
namespace fa2b {

constexpr int kBK = 128;             // keys per unit
constexpr int kDqWarps = 4;
constexpr int kMaxParted = 256;      // key tiles of a row that may come in parts
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
struct Cfg {
  static constexpr int kBQ = D == 256 ? 64 : 128;      // queries per step
  static constexpr int kDH = D < 128 ? D : 128;        // columns of dV, dK and dQ that a unit forms
  static constexpr int kSplit = D / kDH;
  // Step g + 2 takes the buffers of step g crosswise.  dO(g) is done with after dV, early in the step, and leaves its buffer to
  // Q(g + 2), which the next step already wants for its scores; Q(g) is done with at the step's end and leaves its buffer
  // to dO(g + 2).  So both are asked for a step ahead of their use (a load takes 1500 to 2000 cycles beside the reductions)
  // instead of half a step and one and a half.  B2 Hq16 Hkv2 S4096 D256 1433 us without, 1215 with; B4 Hq32 Hkv8 S8192 D64
  // 4117, 4000 to 4066; D 128, whose steps are long enough, 6200 to 6300, 6310 to 6340.
  static constexpr bool kCross = D != 128;
  static constexpr bool kAlias = D >= 128;             // dQ in dP's columns
  static constexpr bool kVTmem = D == 256;             // V in TMEM, as the A operand of dP
  static constexpr bool kTransDq = D == 256;           // dQ^T: lanes are columns of dq, columns are queries
  static constexpr int kDqCols = kTransDq ? kBQ : kDH; // TMEM columns of dQ
  // Softmax warpgroups.  At D 64 the softmax is longer than the products, and four hide each other's latencies better (with dP(t+1)
  // before dQ(t); one without the other gains less or loses).  Two and four, us, 128 queries a tile: B3 Hq12 Hkv4
  // 1000 x 1531 79.5, 73.9; B1 Hq32 Hkv8 S2048 97.5, 94.7; B4 Hq16 Hkv4 S1024 63.3, 60.8; B8 Hq8 S2048 186.5, 185.9; B16 Hq12
  // S512 without mask 103.7, 105.7; B4 Hq32 Hkv8 S8192, at the power limit, 4115, 4178.
  static constexpr int kGroups = D == 64 ? 4 : 2;
  static constexpr int kGroupQ = kBQ / kGroups;        // query columns of one
  static constexpr int kSoftmaxWarps = 4 * kGroups;
  static constexpr int kWarpTma = kSoftmaxWarps + kDqWarps, kWarpMma = kWarpTma + 1, kWarpPass = kWarpTma + 2;
  static constexpr int kThreads = (kWarpTma + 4) * 32;
  static constexpr int kUnitReaders = 3 + kSoftmaxWarps + kDqWarps;
  // registers of the softmax, dQ and other warps, which share those that the CTA is launched with
  static constexpr int kSoftmaxRegs = kGroups == 4 ? 88 : 144, kDqRegs = kGroups == 4 ? 88 : 152,
                       kOtherRegs = kGroups == 4 ? 40 : 64;
  static_assert(kSoftmaxWarps * kSoftmaxRegs + kDqWarps * kDqRegs + 4 * kOtherRegs <= kThreads / 32 * (65536 / kThreads / 8 * 8),
                "registers");
  // Cycles between 8 KB of reductions: an SM sends about 25 bytes a cycle, and reductions that wait for that keep the
  // tensor core from shared memory and TMA requests in the queue (B4 Hq32 Hkv8 S8192: D 128 6809 us without, 6200
  // with 288, 6155 with 304, 6300 with 320, 6623 with 440; D 64 4199 without, 4025 with 320, 4200 with 800; B2 Hq16 Hkv2
  // S4096 D256 1218 without, 1195 with 300, 1215 with 500).  Half as many at half the distance gains nothing.
  static constexpr int kPace = D == 128 ? 304 : D == 64 ? 320 : 300;
  static constexpr uint32_t kColS = 0;
  static constexpr uint32_t kColDp = kBQ;
  static constexpr uint32_t kColDq = kAlias ? kColDp : 2 * kBQ;
  static constexpr uint32_t kColDv = kAlias ? 2 * kBQ : kColDq + kDqCols;
  static constexpr uint32_t kColDk = kColDv + kDH;
  static constexpr uint32_t kColV = kColDk + kDH;
  static_assert(kColV + (kVTmem ? D / 2 : 0) <= 512, "TMEM columns");
  static constexpr int kKBox = kBK * 128;              // 128 keys x 64 columns
  static constexpr int kQBox = kBQ * 128;              // kBQ queries x 64 columns
  static constexpr int kBoxes = kDH / 64;              // boxes of the columns of dV, dK
  static constexpr int kKBytes = (D / 64) * kKBox;
  static constexpr int kQBytes = (D / 64) * kQBox;
  static constexpr int kDsBytes = kBK * kBQ * 2;       // boxes of 128 keys x 64 queries
  static constexpr int kDsBuffers = kAlias ? 1 : 2;    // dP(t + 1), and with it dS(t + 1), does not wait for dQ(t) and dK(t)
  static constexpr int kRowBytes = kBQ * 4;            // lse2 or delta of a query tile
  static constexpr int kK = 0;
  static constexpr int kV = kK + kKBytes;
  static constexpr int kQ = kV + (kVTmem ? 0 : kKBytes);
  static constexpr int kDs = kQ + 4 * kQBytes;         // four buffers of Q and dO, see q_buffer
  static constexpr int kLse = kDs + kDsBuffers * kDsBytes;          // two stages
  static constexpr int kDelta = kLse + 2 * kRowBytes;  // two stages
  static constexpr int kBytes = kDelta + 2 * kRowBytes;
  static_assert(kBytes + 1024 <= 227 * 1024, "shared memory");  // 1024: the barriers, rounded up to the tiles' alignment
};

struct Params {
  __nv_bfloat16 *dq, *dk, *dv;
  const __nv_bfloat16* v;
  long long q_sb, q_sh, q_ss;        // element strides of q, o, do, dq (batch, head, row)
  long long k_sb, k_sh, k_ss;        // and of k, v, dk, dv
  const float* stats;                // [batch * hq][nq][lse2, delta][kBQ]
  int streams;                       // sums that a query tile's dQ is gathered in: key tile j adds to sum j % streams
  float* acc;                        // [streams][batch * hq][nq][split][kDqCols / 4][128][4]
  uint32_t* turns;                   // [streams][batch * hq][nq][split]
  long long tiles;                   // batch * hq * nq * split
  uint32_t* ticket;
  int batch, hq, hkv, group, sq, skv, nq, nk;
  int units;
  int wave;                          // the order of the units, see Unit
  int per_row;                       // units of a row: nk, or with parts first[nk]
  int part_tiles;                    // query tiles of a part
  float* partial;                    // [rows][per_row][dV, dK][kDH / 4][128][4]
  uint16_t first[kMaxParted + 1];    // with parts: the first unit of each key tile in its row
  int causal;
  float scale, scale_log2;
  uint32_t* status;
};

// One unit: key tile j of (b, kvh), column half `half`.  The steps of a key tile visit the query tiles nq-1 .. i_min,
// each for every query head of the group (heads inside tiles: head by head, a later and shorter unit could not
// pass the earlier one into the next head, B2 Hq16 Hkv2 S4096 D256 took 2490 us for 1744).  Where key tiles are too
// few to fill the GPU a unit is one of `parts` parts of a tile's steps, p.part_tiles query tiles each (cut at the same query
// tiles for every key tile: their turns go with each other), and leaves its dV and dK in fp32 for fa2_bwd_finish to
// add.  Units are numbered wave by wave: within a wave of p.wave (b, kvh, half) rows, all
// their first units, then all their second ones, and so on.
struct Unit {
  int b, kvh, j, half;
  int i0, steps;         // first query tile, number of steps
  int parts;
  long long slot;        // of p.partial
};

template <int D>
__device__ __forceinline__ Unit decode_unit(const Params& p, int u) {
  using C = Cfg<D>;
  Unit x;
  const int rows = p.batch * p.hkv * C::kSplit;
  const int first = u / (p.wave * p.per_row) * p.wave;  // first row of the wave
  const int in_wave = min(p.wave, rows - first);
  u -= first * p.per_row;
  const int v = u / in_wave;
  int row = first + u - v * in_wave;
  x.slot = static_cast<long long>(row) * p.per_row + v;
  x.half = row % C::kSplit;
  row /= C::kSplit;
  x.kvh = row % p.hkv;
  x.b = row / p.hkv;
  int part = 0;
  x.j = v;
  x.parts = 1;
  if (p.partial != nullptr) {
    int lo = 0, hi = p.nk;  // first[lo] <= v < first[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (p.first[mid] <= v)
        lo = mid;
      else
        hi = mid;
    }
    x.j = lo;
    part = v - p.first[lo];
    x.parts = p.first[lo + 1] - p.first[lo];
  }
  const int all = max(0, p.nq - (p.causal ? x.j * (kBK / C::kBQ) : 0));  // query tiles
  const int skip = part * p.part_tiles;
  x.i0 = p.nq - 1 - skip;
  x.steps = (x.parts > 1 ? min(p.part_tiles, all - skip) : all) * p.group;
  return x;
}

// The step after (i, h)
__device__ __forceinline__ void next_step(const Params& p, int& i, int& h) {
  if (++h == p.group) {
    h = 0;
    --i;
  }
}

// Buffers of step g's Q and dO: steps g and g + 2 share a pair.
template <int D>
__device__ __forceinline__ int q_buffer(int g) {
  return (g & 1) * 2 + (Cfg<D>::kCross ? (g >> 1) & 1 : 0);
}
template <int D>
__device__ __forceinline__ int do_buffer(int g) {
  return q_buffer<D>(g) ^ 1;
}

// number of key tiles that add to query tile i
template <int D>
__device__ __forceinline__ int contributors(const Params& p, int i) {
  if (!p.causal) return p.nk;
  return min(p.nk, (min((i + 1) * Cfg<D>::kBQ, p.sq) - 1) / kBK + 1);
}

// One lane of the (whole) warp, the same on every call.
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(is));
  return is != 0;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void red_add_v4(float* dst, float a, float b, float c, float d) {
  asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(dst), "f"(a), "f"(b), "f"(c), "f"(d)
               : "memory");
}

// Waits (bounded) until the turn counter reads `want`.
__device__ __forceinline__ bool wait_turn(const uint32_t* turn, uint32_t want, uint32_t* status) {
  const unsigned long long t0 = global_timer_ns();
  while (true) {
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(turn) : "memory");
    if (v == want) return true;
    if (cta_abort_flag() != 0u) return false;
    if (global_timer_ns() - t0 > kWaitTimeoutNs) {
      record_status(status, kDevTimeoutPipe);
      cta_abort_flag() = 1u;
      return false;
    }
    __nanosleep(20);
  }
}

// 16 lanes x 8 N columns of TMEM, dealt out like an mma accumulator: thread l gets, of every 8 columns i,
// r[4i], r[4i+1] = columns 2 (l % 4), + 1 of lane l / 4 and r[4i+2], r[4i+3] the same of lane l / 4 + 8.
// No wait.
template <int N>
__device__ __forceinline__ void tmem_ld_frag(uint32_t a, uint32_t* r) {
  static_assert(N == 4 || N == 8, "groups of columns");
  if constexpr (N == 8) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(a)
        : "memory");
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(a)
        : "memory");
  }
}

// The counterpart for values packed in pairs: 16 lanes x 4 N 32-bit columns, r[2i] of lane l / 4, r[2i+1] of
// lane l / 4 + 8, column 4 i + l % 4.
template <int N>
__device__ __forceinline__ void tmem_st_frag(uint32_t a, const uint32_t* r) {
  static_assert(N == 4 || N == 8, "groups of columns");
  if constexpr (N == 8) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(a),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
  } else {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"r"(a), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  }
}

__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Four 8 x 8 matrices of 16-bit values from such a layout to shared memory; lane l gives the address
// of row l % 8 of matrix l / 8.
__device__ __forceinline__ void st_matrix_x4(uint32_t addr, const uint32_t* r) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3])
               : "memory");
}

template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&r)[N]) {
  static_assert(N == 64 || N == 128, "columns");
  if constexpr (N == 64) {
    tmem_ld64(addr, r);
  } else {
    tmem_ld64(addr, *reinterpret_cast<uint32_t(*)[64]>(&r[0]));
    tmem_ld64(addr + 64, *reinterpret_cast<uint32_t(*)[64]>(&r[64]));
  }
}

template <int D>
__global__ void __launch_bounds__(Cfg<D>::kThreads, 1)
    fa2_bwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                   const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p) {
  using C = Cfg<D>;
  extern __shared__ __align__(1024) uint8_t smem[];  // no room is left to round its start up
  __shared__ uint64_t bar_unit_full[2], bar_unit_empty[2], bar_kv_full, bar_kv_empty, bar_v, bar_q_full[2], bar_q_empty[2],
      bar_do_full[2], bar_do_empty[2], bar_s, bar_p, bar_dp, bar_ds, bar_dq, bar_dqfree, bar_turn[2], bar_added[2],
      bar_passed[2], bar_acc, bar_accfree, bar_drain;
  __shared__ int unit_ring[2];
  __shared__ uint32_t tmem_base_shared;

  const int warp = warp_id();
  const int lane = lane_id();
  if ((smem_u32(smem) & 1023u) != 0u) {  // the swizzled tiles would lie wrong
    if (threadIdx.x == 0) record_status(p.status, kDevBadArgs);
    return;
  }

  if (threadIdx.x == 0) {
    cta_abort_flag() = 0u;
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_unit_full[i], 1);
      mbar_init(&bar_unit_empty[i], C::kUnitReaders);
      mbar_init(&bar_q_full[i], 1);
      mbar_init(&bar_q_empty[i], 1);
      mbar_init(&bar_do_full[i], 1);
      mbar_init(&bar_do_empty[i], 1);
      mbar_init(&bar_turn[i], 1);
      mbar_init(&bar_added[i], kDqWarps);
      mbar_init(&bar_passed[i], 1);
    }
    mbar_init(&bar_kv_full, 1);
    mbar_init(&bar_kv_empty, 1);
    mbar_init(&bar_v, C::kSoftmaxWarps);
    mbar_init(&bar_s, 1);
    mbar_init(&bar_p, C::kSoftmaxWarps);
    mbar_init(&bar_dp, 1);
    mbar_init(&bar_ds, C::kSoftmaxWarps);
    mbar_init(&bar_dq, 1);
    mbar_init(&bar_dqfree, kDqWarps);
    mbar_init(&bar_acc, 1);
    mbar_init(&bar_accfree, C::kSoftmaxWarps);
    mbar_init(&bar_drain, 1);
    fence_barrier_init();
  }
  if (warp == C::kWarpMma) {
    tmem_alloc(&tmem_base_shared, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = tmem_base_shared;
  wait_previous_kernels();

  // The r-th unit of this CTA (-1: no more), for the one thread or the warp that reads the ring.
  auto next_unit = [&](int r, bool& ok) -> int {
    if (!mbar_wait(&bar_unit_full[r & 1], (r >> 1) & 1, p.status, kDevTimeoutPipe)) {
      ok = false;
      return -1;
    }
    return *reinterpret_cast<volatile int*>(&unit_ring[r & 1]);
  };

  if (warp >= C::kWarpTma) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));
    if (warp == C::kWarpTma) {
      // ---------------------------------------------------------------- unit counter, TMA
      if (lane == 0) {
        tma_prefetch_desc(&map_q);
        tma_prefetch_desc(&map_do);
        tma_prefetch_desc(&map_k);
        tma_prefetch_desc(&map_v);
        asm volatile("fence.proxy.async.global;" ::: "memory");  // the statistics of the launch before
        bool ok = true;
        int g = 0;       // steps begun
        int loads = 0;   // units whose K and V were loaded
        int q_issued = 0, do_issued = 0;
        for (int r = 0; ok; ++r) {
          if (r >= 2 && !mbar_wait(&bar_unit_empty[r & 1], ((r >> 1) - 1) & 1, p.status, kDevTimeoutPipe)) break;
          const uint32_t tk = atomicAdd(p.ticket, 1u);
          const int u = tk < static_cast<uint32_t>(p.units) ? static_cast<int>(tk) : -1;
          *reinterpret_cast<volatile int*>(&unit_ring[r & 1]) = u;
          mbar_arrive(&bar_unit_full[r & 1]);
          if (u < 0) break;
          const Unit x = decode_unit<D>(p, u);
          {
            int i = x.i0, h = 0;
            for (int t = 0; t < x.steps; ++t, ++g, next_step(p, i, h)) {
              const int head = x.kvh * p.group + h;
              const long long bh = static_cast<long long>(x.b) * p.hq + head;
              const int st = g & 1;
              if (g >= 2 && !mbar_wait(&(C::kCross ? bar_do_empty : bar_q_empty)[st], ((g >> 1) - 1) & 1, p.status, kDevTimeoutPipe)) {
                ok = false;
                break;
              }
              mbar_arrive_expect_tx(&bar_q_full[st], C::kQBytes + C::kRowBytes);
              for (int bx = 0; bx < D / 64; ++bx)
                tma_load_4d(smem + C::kQ + q_buffer<D>(g) * C::kQBytes + bx * C::kQBox, &map_q, &bar_q_full[st], bx * 64, i * C::kBQ,
                            head, x.b);
              const float* rows = p.stats + (bh * p.nq + i) * (2 * C::kBQ);
              bulk_load(smem + C::kLse + st * C::kRowBytes, rows, C::kRowBytes, &bar_q_full[st]);
              q_issued = g + 1;
              if (t == 0) {
                if (loads > 0 && !mbar_wait(&bar_kv_empty, (loads - 1) & 1, p.status, kDevTimeoutPipe)) {
                  ok = false;
                  break;
                }
                mbar_arrive_expect_tx(&bar_kv_full, (C::kVTmem ? 1 : 2) * C::kKBytes);
                for (int bx = 0; bx < D / 64; ++bx)
                  tma_load_4d(smem + C::kK + bx * C::kKBox, &map_k, &bar_kv_full, bx * 64, x.j * kBK, x.kvh, x.b);
                for (int bx = 0; !C::kVTmem && bx < D / 64; ++bx)
                  tma_load_4d(smem + C::kV + bx * C::kKBox, &map_v, &bar_kv_full, bx * 64, x.j * kBK, x.kvh, x.b);
                ++loads;
              }
              if (g >= 2 && !mbar_wait(&(C::kCross ? bar_q_empty : bar_do_empty)[st], ((g >> 1) - 1) & 1, p.status, kDevTimeoutPipe)) {
                ok = false;
                break;
              }
              mbar_arrive_expect_tx(&bar_do_full[st], C::kQBytes + C::kRowBytes);
              for (int bx = 0; bx < D / 64; ++bx)
                tma_load_4d(smem + C::kQ + do_buffer<D>(g) * C::kQBytes + bx * C::kQBox, &map_do, &bar_do_full[st], bx * 64,
                            i * C::kBQ, head, x.b);
              bulk_load(smem + C::kDelta + st * C::kRowBytes, rows + C::kBQ, C::kRowBytes, &bar_do_full[st]);
              do_issued = g + 1;
            }
          }
        }
        // before the CTA retires, let the last loads land (bounded; a no-op on the normal path)
        if (loads > 0) mbar_drain(&bar_kv_full, (loads - 1) & 1);
        for (int t = max(0, q_issued - 2); t < q_issued; ++t) mbar_drain(&bar_q_full[t & 1], (t >> 1) & 1);
        for (int t = max(0, do_issued - 2); t < do_issued; ++t) mbar_drain(&bar_do_full[t & 1], (t >> 1) & 1);
      }
      __syncwarp();
    } else if (warp == C::kWarpMma) {
      // ---------------------------------------------------------------- MMA issuer
      // The whole warp walks the steps and waits, one elected lane issues: so addresses and
      // descriptors are warp-uniform (issued from a branch of one lane, an MMA took 75 to 135 cycles
      // instead of the tensor core's 64, D 128).
      constexpr uint32_t idesc_s = make_idesc(kBK, C::kBQ, 1, 0, 0);
      constexpr uint32_t idesc_kv = make_idesc(kBK, C::kDH, 1, 0, 1);
      constexpr uint32_t idesc_dq = C::kTransDq ? make_idesc(C::kDH, C::kBQ, 1, 1, 1) : make_idesc(C::kBQ, C::kDH, 1, 1, 1);
      const uint32_t tb = __shfl_sync(0xffffffffu, tbase, 0);
      const uint32_t base = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
      const bool leader = elect_one();
      const uint32_t k_addr = base + C::kK, v_addr = base + C::kV;
      const uint32_t q_base = base + C::kQ;
      // X^T = A B^T over head_dim: S^T = K Q^T, dP^T = V dO^T (all K-major)
      auto issue_scores = [&](uint32_t a, uint32_t b, uint32_t col) {
        const uint64_t ad = make_sdesc_sw128(a, 16, 1024), bd = make_sdesc_sw128(b, 16, 1024);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_bf16_ss(tb + col, ad + (((kk >> 2) * C::kKBox + (kk & 3) * 32) >> 4), bd + (((kk >> 2) * C::kQBox + (kk & 3) * 32) >> 4),
                       idesc_s, kk > 0 ? 1u : 0u);
      };
      // the same with V in TMEM
      auto issue_dp_tmem = [&](uint32_t b) {
        const uint64_t bd = make_sdesc_sw128(b, 16, 1024);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_bf16_ts(tb + C::kColDp, tb + C::kColV + kk * 8, bd + (((kk >> 2) * C::kQBox + (kk & 3) * 32) >> 4), idesc_s,
                       kk > 0 ? 1u : 0u);
      };
      bool ok = true;
      int g = 0;          // steps of earlier units
      int active = 0;     // earlier units with steps (K/V and accumulator phases)
      auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
        return static_cast<bool>(__all_sync(0xffffffffu, mbar_wait(bar, parity, p.status, code)));
      };
      for (int r = 0; ok; ++r) {
        const int u = __shfl_sync(0xffffffffu, next_unit(r, ok), 0);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok || u < 0) break;
        if (leader) mbar_arrive(&bar_unit_empty[r & 1]);
        const Unit x = decode_unit<D>(p, u);
        if (x.steps == 0) continue;
        const uint32_t half_k = x.half * (C::kDH / 64) * C::kKBox, half_q = x.half * (C::kDH / 64) * C::kQBox;
        auto issue_s = [&](int gs) -> bool {
          if (!wait(&bar_q_full[gs & 1], (gs >> 1) & 1, kDevTimeoutTma)) return false;
          tc_fence_after();
          if (leader) {
            issue_scores(k_addr, q_base + q_buffer<D>(gs) * C::kQBytes, C::kColS);
            umma_commit(&bar_s);
          }
          __syncwarp();
          return true;
        };
        auto issue_dp = [&](int gs) {
          if (leader) {
            const uint32_t b = q_base + do_buffer<D>(gs) * C::kQBytes;
            if constexpr (C::kVTmem)
              issue_dp_tmem(b);
            else
              issue_scores(v_addr, b, C::kColDp);
            umma_commit(&bar_dp);
          }
          __syncwarp();
        };
        ok = wait(&bar_kv_full, active & 1, kDevTimeoutTma) && issue_s(g);
        for (int t = 0; ok && t < x.steps; ++t) {
          const int gt = g + t, st = gt & 1;
          const uint32_t q_addr = q_base + q_buffer<D>(gt) * C::kQBytes, do_addr = q_base + do_buffer<D>(gt) * C::kQBytes;
          // dP(t); at D >= 128 its columns hold dQ(t-1) until the dQ warps have read it, at D 64 it was issued in front of
          // dQ(t-1)
          if (C::kAlias || t == 0) {
            ok = wait(&bar_do_full[st], (gt >> 1) & 1, kDevTimeoutTma) &&
                 (!C::kAlias || gt == 0 || wait(&bar_dqfree, (gt - 1) & 1, kDevTimeoutPipe)) &&
                 (!C::kVTmem || t > 0 || wait(&bar_v, active & 1, kDevTimeoutPipe));
            if (!ok) break;
            tc_fence_after();
            issue_dp(gt);
          }
          // dV += P^T dO; the first overwrites an accumulator that the previous unit's epilogue has read
          ok = wait(&bar_p, gt & 1, kDevTimeoutPipe) &&
               (t > 0 || active == 0 || wait(&bar_accfree, (active - 1) & 1, kDevTimeoutPipe));
          if (!ok) break;
          tc_fence_after();
          if (leader) {
            const uint64_t bd = make_sdesc_sw128(do_addr + half_q, C::kQBox, 1024);
#pragma unroll
            for (int kk = 0; kk < C::kBQ / 16; ++kk) {
              constexpr int per = C::kGroupQ / 16;  // steps in a warpgroup's part of P
              umma_bf16_ts(tb + C::kColDv, tb + C::kColS + (kk / per) * C::kGroupQ + (kk % per) * 8, bd + ((kk * 2048) >> 4),
                           idesc_kv, (t > 0 || kk > 0) ? 1u : 0u);
            }
            umma_commit(&bar_do_empty[st]);
          }
          __syncwarp();
          if (t + 1 < x.steps) {
            ok = issue_s(gt + 1);
            if (!ok) break;
          }
          ok = wait(&bar_ds, gt & 1, kDevTimeoutPipe);
          if (!ok) break;
          if constexpr (!C::kAlias) {
            if (t + 1 < x.steps) {
              ok = wait(&bar_do_full[st ^ 1], ((gt + 1) >> 1) & 1, kDevTimeoutTma);
              if (!ok) break;
              tc_fence_after();
              issue_dp(gt + 1);
            }
            ok = gt == 0 || wait(&bar_dqfree, (gt - 1) & 1, kDevTimeoutPipe);
            if (!ok) break;
          }
          tc_fence_after();
          if (leader) {
            const uint32_t ds_addr = base + C::kDs + (C::kDsBuffers == 2 ? st * C::kDsBytes : 0);
            // dQ = dS K (or its transpose)
            const uint64_t dsd = make_sdesc_sw128(ds_addr, C::kKBox, 1024);
            const uint64_t kd = make_sdesc_sw128(k_addr + half_k, C::kKBox, 1024);
#pragma unroll
            for (int kk = 0; kk < kBK / 16; ++kk)
              umma_bf16_ss(tb + C::kColDq, (C::kTransDq ? kd : dsd) + ((kk * 2048) >> 4),
                           (C::kTransDq ? dsd : kd) + ((kk * 2048) >> 4), idesc_dq, kk > 0 ? 1u : 0u);
            umma_commit(&bar_dq);
            // dK += dS^T Q
            const uint64_t dsk = make_sdesc_sw128(ds_addr, 16, 1024);
            const uint64_t qd = make_sdesc_sw128(q_addr + half_q, C::kQBox, 1024);
#pragma unroll
            for (int kk = 0; kk < C::kBQ / 16; ++kk)
              umma_bf16_ss(tb + C::kColDk, dsk + (((kk >> 2) * C::kKBox + (kk & 3) * 32) >> 4), qd + ((kk * 2048) >> 4), idesc_kv,
                           (t > 0 || kk > 0) ? 1u : 0u);
            umma_commit(&bar_q_empty[st]);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (leader) {
          umma_commit(&bar_acc);
          umma_commit(&bar_kv_empty);
        }
        __syncwarp();
        g += x.steps;
        ++active;
      }
      // every MMA issued completes before TMEM is released (bounded)
      if (leader) {
        umma_commit(&bar_drain);
        mbar_drain(&bar_drain, 0);
      }
      __syncwarp();
    } else if (lane == 0) {
      // ---------------------------------------------------------------- turns of the dQ sums
      // The last warp waits for a step's turn, a step or two ahead of the dQ warps' additions; kWarpPass waits for
      // those, for their arrival in L2 (the fence: 1700 cycles, which the dQ warps need not stand still for),
      // and passes the turn on.
      const bool pass = warp == C::kWarpPass;
      bool ok = true;
      int g = 0;
      for (int r = 0; ok; ++r) {
        const int u = next_unit(r, ok);
        if (!ok || u < 0) break;
        mbar_arrive(&bar_unit_empty[r & 1]);
        if (p.nk == 1) continue;  // no sums
        const Unit x = decode_unit<D>(p, u);
        uint32_t* turns = p.turns + x.j % p.streams * p.tiles;
        const uint32_t rank = x.j / p.streams;
        {
          int i = x.i0, h = 0;
          for (int t = 0; t < x.steps; ++t, ++g, next_step(p, i, h)) {
            const int count = contributors<D>(p, i);
            const long long bh = static_cast<long long>(x.b) * p.hq + x.kvh * p.group + h;
            uint32_t* turn = turns + (bh * p.nq + i) * C::kSplit + x.half;
            if (pass) {
              ok = mbar_wait(&bar_added[g & 1], (g >> 1) & 1, p.status, kDevTimeoutPipe);
              if (!ok) break;
              if (x.j + p.streams < count) {
                __threadfence();
                asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(turn), "r"(rank + 1) : "memory");
              }
              mbar_arrive(&bar_passed[g & 1]);
            } else {
              ok = (g < 2 || mbar_wait(&bar_passed[g & 1], ((g >> 1) - 1) & 1, p.status, kDevTimeoutPipe)) &&
                   (rank == 0 || wait_turn(turn, rank, p.status));
              if (!ok) break;
              mbar_arrive(&bar_turn[g & 1]);
            }
          }
        }
      }
    }
  } else if (warp >= C::kSoftmaxWarps) {
    // ------------------------------------------------------------------ dQ: TMEM -> global, in turn
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kDqRegs));
    const int wq = warp & 3;
    const int row = wq * 32 + lane;  // TMEM lane: a query of the tile, or (transposed) a column of dq
    const uint32_t col = tmem_addr(tbase, wq * 32, C::kColDq);
    bool ok = true;
    int g = 0;
    for (int r = 0; ok; ++r) {
      const int u = __shfl_sync(0xffffffffu, lane == 0 ? next_unit(r, ok) : 0, 0);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok || u < 0) break;
      if (lane == 0) mbar_arrive(&bar_unit_empty[r & 1]);
      const Unit x = decode_unit<D>(p, u);
      {
        int i = x.i0, h = 0;
        for (int t = 0; t < x.steps; ++t, ++g, next_step(p, i, h)) {
          const int head = x.kvh * p.group + h;
          const long long bh = static_cast<long long>(x.b) * p.hq + head;
          const long long tile = (bh * p.nq + i) * C::kSplit + x.half;
          if (!__all_sync(0xffffffffu, mbar_wait(&bar_dq, g & 1, p.status, kDevTimeoutMma))) {
            ok = false;
            break;
          }
          tc_fence_after();
          uint32_t v[C::kDqCols];
          tmem_load(col, v);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_dqfree);
          float* acc = p.acc + (x.j % p.streams * p.tiles + tile) * (C::kDqCols * 128) + row * 4;
          if (p.nk > 1) {
            if (!__all_sync(0xffffffffu, mbar_wait(&bar_turn[g & 1], (g >> 1) & 1, p.status, kDevTimeoutPipe))) {
              ok = false;
              break;
            }
            if (x.j < p.streams) {
#pragma unroll
              for (int c = 0; c < C::kDqCols / 4; ++c)
                __stcg(reinterpret_cast<float4*>(acc + c * 512),
                       make_float4(__uint_as_float(v[4 * c]), __uint_as_float(v[4 * c + 1]), __uint_as_float(v[4 * c + 2]),
                                   __uint_as_float(v[4 * c + 3])));
            } else {
#pragma unroll
              for (int c = 0; c < C::kDqCols / 4; ++c) {
                if (c % 4 == 0 && c > 0)
                  for (const long long t0 = clock64(); clock64() - t0 < C::kPace;) {}
                red_add_v4(acc + c * 512, __uint_as_float(v[4 * c]), __uint_as_float(v[4 * c + 1]),
                           __uint_as_float(v[4 * c + 2]), __uint_as_float(v[4 * c + 3]));
              }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_added[g & 1]);
          } else {  // one key tile: the sum is complete
            __nv_bfloat16* out = p.dq + x.b * p.q_sb + head * p.q_sh + static_cast<long long>(i) * C::kBQ * p.q_ss +
                                 x.half * C::kDH;
            const int rows = min(C::kBQ, p.sq - i * C::kBQ);
            if constexpr (C::kTransDq) {
#pragma unroll
              for (int q = 0; q < C::kDqCols; ++q)
                if (q < rows) out[q * p.q_ss + row] = __float2bfloat16_rn(__uint_as_float(v[q]) * p.scale);
            } else if (row < rows) {
              uint4* dst = reinterpret_cast<uint4*>(out + row * p.q_ss);
#pragma unroll
              for (int c = 0; c < C::kDqCols / 8; ++c) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  w[e] = pack_bf16x2(__uint_as_float(v[8 * c + 2 * e]) * p.scale, __uint_as_float(v[8 * c + 2 * e + 1]) * p.scale);
                dst[c] = make_uint4(w[0], w[1], w[2], w[3]);
              }
            }
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax warps, epilogue of dV and dK
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
    const int wg = warp >> 2;
    const int row = (warp & 3) * 32 + lane;  // key of the tile
    const uint32_t lanes = tmem_addr(tbase, (warp & 3) * 32, 0);
    const uint32_t col_s = lanes + C::kColS + wg * C::kGroupQ;
    const uint32_t col_dp = lanes + C::kColDp + wg * C::kGroupQ;
    constexpr int kCols8 = C::kGroupQ / 8;  // groups of 8 query columns
    // this lane's row and first piece in the matrices it stores: matrix l / 8 is the lower (upper) 8 keys of 16
    // in an even (odd) group of 8 queries
    const uint32_t ds_base = smem_u32(smem + C::kDs + wg * C::kGroupQ / 64 * C::kKBox);
    const int st_row = (warp & 3) * 32 + ((lane >> 3) & 1) * 8 + (lane & 7);
    const int st_piece = (lane >> 4) + wg * C::kGroupQ % 64 / 8;
    const F2 c2 = pair2(__float_as_uint(p.scale_log2), __float_as_uint(p.scale_log2));
    // epilogue: the warpgroups that share a box of the dS buffer, the boxes in use at once, lanes that store a row
    constexpr int kSharers = 64 / C::kGroupQ, kSets = C::kGroups / kSharers, kRounds = 2 * C::kBoxes / kSets;
    constexpr int kRowLanes = C::kGroupQ / 8;
    const int set = wg / kSharers, first_col = wg * C::kGroupQ % 64;
    bool ok = true;
    int g = 0, active = 0;
    for (int r = 0;; ++r) {
      const int u = __shfl_sync(0xffffffffu, lane == 0 ? next_unit(r, ok) : 0, 0);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok || u < 0) break;
      if (lane == 0) mbar_arrive(&bar_unit_empty[r & 1]);
      const Unit x = decode_unit<D>(p, u);
      const int key = x.j * kBK + row;
      const bool ragged = x.j * kBK + kBK > p.skv;  // keys behind the last one
      if (C::kVTmem && x.steps > 0) {
        // this warpgroup's half of V's columns, a row per thread; the previous unit's MMAs are complete (bar_acc)
        const uint4* src = reinterpret_cast<const uint4*>(p.v + x.b * p.k_sb + x.kvh * p.k_sh + key * p.k_ss + wg * (D / 2));
#pragma unroll
        for (int part = 0; part < D / 128; ++part) {
          uint32_t v[32];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint4 w = key < p.skv ? __ldg(src + part * 8 + e) : make_uint4(0u, 0u, 0u, 0u);
            v[4 * e] = w.x;
            v[4 * e + 1] = w.y;
            v[4 * e + 2] = w.z;
            v[4 * e + 3] = w.w;
          }
          tmem_st32(lanes + C::kColV + wg * (D / 4) + part * 32, v);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_v);
      }
      {
        int i = x.i0, h = 0;
        for (int t = 0; t < x.steps; ++t, ++g, next_step(p, i, h)) {
          if (!__all_sync(0xffffffffu, mbar_wait(&bar_q_full[g & 1], (g >> 1) & 1, p.status, kDevTimeoutTma) &&
                                           mbar_wait(&bar_s, g & 1, p.status, kDevTimeoutMma))) {
            ok = false;
            break;
          }
          tc_fence_after();
          // this lane's two query columns of every group of 8
          const F2* lse2 = reinterpret_cast<const F2*>(smem + C::kLse + (g & 1) * C::kRowBytes) + wg * (C::kGroupQ / 2) + (lane & 3);
          const F2* delta = lse2 + C::kBQ;  // behind both stages of lse2
          const int q0 = i * C::kBQ + wg * C::kGroupQ;
          const bool masked = ragged || (p.causal && q0 < x.j * kBK + kBK - 1);
          // fragment (h16, rg): key (warp & 3) * 32 + h16 * 16 + rg * 8 + lane / 4
          const int key0 = x.j * kBK + (warp & 3) * 32 + (lane >> 2);
          uint32_t raw[2][4 * kCols8];
          tmem_ld_frag<kCols8>(col_s, raw[0]);
          tmem_ld_frag<kCols8>(col_s + (16u << 16), raw[1]);
          float pr[2][4 * kCols8];
          F2 st[kCols8];
#pragma unroll
          for (int n = 0; n < kCols8; ++n) st[n] = lse2[4 * n];
          tmem_wait_ld();
#pragma unroll
          for (int h16 = 0; h16 < 2; ++h16) {
#pragma unroll
            for (int n = 0; n < kCols8; ++n) {
#pragma unroll
              for (int rg = 0; rg < 2; ++rg) {
                const int e = 4 * n + 2 * rg;
                const float2 x = split2(fma2(pair2(raw[h16][e], raw[h16][e + 1]), c2, st[n]));
                pr[h16][e] = ex2_approx(x.x);
                pr[h16][e + 1] = ex2_approx(x.y);
              }
            }
            if (masked) {
#pragma unroll
              for (int rg = 0; rg < 2; ++rg) {
                const int key = key0 + h16 * 16 + rg * 8;
                // query columns before `first` are masked for this key
                const int first = (key >= p.skv ? C::kGroupQ : (p.causal ? key - q0 : 0)) - 2 * (lane & 3);
#pragma unroll
                for (int n = 0; n < kCols8; ++n) {
                  if (8 * n < first) pr[h16][4 * n + 2 * rg] = 0.0f;
                  if (8 * n + 1 < first) pr[h16][4 * n + 2 * rg + 1] = 0.0f;
                }
              }
            }
            uint32_t packed[2 * kCols8];
#pragma unroll
            for (int e = 0; e < 2 * kCols8; ++e) packed[e] = pack_bf16x2(pr[h16][2 * e], pr[h16][2 * e + 1]);
            tmem_st_frag<kCols8>(col_s + (static_cast<uint32_t>(h16 * 16) << 16), packed);
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_p);
          if (!__all_sync(0xffffffffu, mbar_wait(&bar_do_full[g & 1], (g >> 1) & 1, p.status, kDevTimeoutTma))) {
            ok = false;
            break;
          }
#pragma unroll
          for (int n = 0; n < kCols8; ++n) st[n] = delta[4 * n];
          if (!__all_sync(0xffffffffu, mbar_wait(&bar_dp, g & 1, p.status, kDevTimeoutMma))) {
            ok = false;
            break;
          }
          tc_fence_after();
          tmem_ld_frag<kCols8>(col_dp, raw[0]);
          tmem_ld_frag<kCols8>(col_dp + (16u << 16), raw[1]);
          tmem_wait_ld();
#pragma unroll
          for (int h16 = 0; h16 < 2; ++h16) {
            float ds[4 * kCols8];
#pragma unroll
            for (int n = 0; n < kCols8; ++n) {
#pragma unroll
              for (int rg = 0; rg < 2; ++rg) {
                const int e = 4 * n + 2 * rg;
                const float2 x = split2(mul2(pair2(__float_as_uint(pr[h16][e]), __float_as_uint(pr[h16][e + 1])),
                                             add2(pair2(raw[h16][e], raw[h16][e + 1]), st[n])));
                ds[e] = x.x;
                ds[e + 1] = x.y;
              }
            }
            if (masked) {  // dP may be infinite or NaN there
#pragma unroll
              for (int rg = 0; rg < 2; ++rg) {
                const int key = key0 + h16 * 16 + rg * 8;
                const int first = (key >= p.skv ? C::kGroupQ : (p.causal ? key - q0 : 0)) - 2 * (lane & 3);
#pragma unroll
                for (int n = 0; n < kCols8; ++n) {
                  if (8 * n < first) ds[4 * n + 2 * rg] = 0.0f;
                  if (8 * n + 1 < first) ds[4 * n + 2 * rg + 1] = 0.0f;
                }
              }
            }
#pragma unroll
            for (int n = 0; n < kCols8; n += 2) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(ds[4 * n + 2 * e], ds[4 * n + 2 * e + 1]);
              st_matrix_x4(ds_base + (C::kDsBuffers == 2 ? (g & 1) * C::kDsBytes : 0) +
                               sw128_offset(st_row + h16 * 16, (st_piece + n) * 16),
                           w);
            }
          }
          fence_async_smem();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_ds);
        }
      }
      if (!ok) break;
      // Epilogue: dV and dK, 64 columns at a time.  A warp turns its 32 keys round in its own rows of the dS buffer (the MMAs
      // that read it are complete) and stores rows of 128 bytes (64 where two warpgroups share a box).  With two boxes of dS
      // one half of the warpgroups takes dV and the other dK; with one all take both.  TMA stores from there waited in
      // the TMA unit behind the next unit's loads, 3500 ns a unit at D 128; rows written by their threads, 16 bytes at a
      // stride, took 9600 cycles.  One tile of 128 14.1 us with TMA stores, 12.3 so; B3 Hq12 Hkv4 1000 x 1531 D64 73.6, 71.8;
      // B4 Hq16 Hkv4 S1024 D128 90.8, 89.
      if (x.steps > 0 && !__all_sync(0xffffffffu, mbar_wait(&bar_acc, active & 1, p.status, kDevTimeoutMma))) break;
      tc_fence_after();
      if (x.parts > 1) {  // a part: fp32, as fa2_bwd_finish reads it
        constexpr int kPerSum = C::kGroups / 2, kCols = C::kDH / kPerSum;
        float* dst = p.partial + (x.slot * 2 + wg / kPerSum) * (C::kDH * 128) + row * 4;
#pragma unroll 1
        for (int dc = wg % kPerSum * kCols; dc < (wg % kPerSum + 1) * kCols; dc += 32) {
          uint32_t a[32];
          tmem_ld32(lanes + (wg / kPerSum == 0 ? C::kColDv : C::kColDk) + dc, a);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            __stcg(reinterpret_cast<float4*>(dst + (dc / 4 + e) * 512),
                   make_float4(__uint_as_float(a[4 * e]), __uint_as_float(a[4 * e + 1]), __uint_as_float(a[4 * e + 2]),
                               __uint_as_float(a[4 * e + 3])));
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_accfree);
        ++active;
        continue;
      }
      for (int round = 0; round < kRounds; ++round) {
        const int which = kSets == 2 ? set : round / C::kBoxes;  // 0: dV, 1: dK
        const int box = kSets == 2 ? round : round % C::kBoxes;
        const float mul = which == 0 ? 1.0f : p.scale;
        const uint32_t from = lanes + (which == 0 ? C::kColDv : C::kColDk) + box * 64 + wg % kSharers * C::kGroupQ;
        uint32_t a[2][4 * kCols8];
        if (x.steps > 0) {
          tmem_ld_frag<kCols8>(from, a[0]);
          tmem_ld_frag<kCols8>(from + (16u << 16), a[1]);
          tmem_wait_ld();
        } else {  // a tile that no query sees
#pragma unroll
          for (int e = 0; e < 4 * kCols8; ++e) a[0][e] = a[1][e] = 0u;
        }
#pragma unroll
        for (int h16 = 0; h16 < 2; ++h16) {
#pragma unroll
          for (int n = 0; n < kCols8; n += 2) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = pack_bf16x2(__uint_as_float(a[h16][4 * n + 2 * e]) * mul, __uint_as_float(a[h16][4 * n + 2 * e + 1]) * mul);
            st_matrix_x4(ds_base + sw128_offset(st_row + h16 * 16, (st_piece + n) * 16), w);
          }
        }
        if (round == kRounds - 1 && x.steps > 0) {  // the accumulators are read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_accfree);
          ++active;
        }
        __syncwarp();
        uint4 w[kRowLanes];
#pragma unroll
        for (int e = 0; e < kRowLanes; ++e)
          w[e] = *reinterpret_cast<const uint4*>(
              smem + C::kDs + set * C::kKBox +
              sw128_offset((warp & 3) * 32 + (e * 32 + lane) / kRowLanes, first_col * 2 + lane % kRowLanes * 16));
        __nv_bfloat16* out = (which == 0 ? p.dv : p.dk) + x.b * p.k_sb + x.kvh * p.k_sh + x.half * C::kDH + box * 64 + first_col +
                             lane % kRowLanes * 8;
#pragma unroll
        for (int e = 0; e < kRowLanes; ++e) {
          const int key = x.j * kBK + (warp & 3) * 32 + (e * 32 + lane) / kRowLanes;
          if (key < p.skv) *reinterpret_cast<uint4*>(out + key * p.k_ss) = w[e];
        }
        __syncwarp();
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == C::kWarpMma) {
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

// delta = sum do * o and lse * log2(e) of every row, both negated, in rows padded to whole query tiles; D / 8
// lanes a row, 16 bytes a lane, four rows a thread.  Also sets the unit counter and the turn counters to 0.
// A block lies in one query tile, so that the divisions are its own and not, in 64 bits, each row's (67 MB read in 18 us so, in
// 13.7 now; 537 MB in 85).
template <int D>
struct Prep {
  static constexpr int kLanes = D / 8, kPass = 256 / kLanes, kRows = 4 * kPass;  // lanes a row, rows a pass, rows a block
  static constexpr int kBlocks = Cfg<D>::kBQ / kRows;                            // blocks a query tile
  static_assert(kBlocks * kRows == Cfg<D>::kBQ, "blocks");
};

template <int D>
__global__ void __launch_bounds__(256) fa2_bwd_prep(const __nv_bfloat16* __restrict__ o, const __nv_bfloat16* __restrict__ dout,
                                                    const float* __restrict__ lse, float* __restrict__ stats,
                                                    uint32_t* __restrict__ counters, long long n_counters, int sq, int nq, int hq,
                                                    long long sb, long long sh, long long ss) {
  using C = Cfg<D>;
  using R = Prep<D>;
  allow_next_kernel();
  const uint32_t tile = blockIdx.x / R::kBlocks;  // (b * hq + h) * nq + query tile
  const uint32_t bh = tile / static_cast<uint32_t>(nq), b = bh / static_cast<uint32_t>(hq);
  const int in_tile = static_cast<int>(blockIdx.x % R::kBlocks) * R::kRows + static_cast<int>(threadIdx.x) / R::kLanes;
  const int first = static_cast<int>(tile - bh * nq) * C::kBQ + in_tile;
  const int part = threadIdx.x % R::kLanes;
  const long long off = b * sb + (bh - b * hq) * sh + first * ss + part * 8;
  wait_previous_kernels();
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < n_counters; i += static_cast<long long>(gridDim.x) * 256)
    counters[i] = 0u;
  uint4 x[4], y[4];
  float l[4], sum[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int i = first + n * R::kPass;
    x[n] = i < sq ? *reinterpret_cast<const uint4*>(o + off + n * R::kPass * ss) : make_uint4(0u, 0u, 0u, 0u);
    y[n] = i < sq ? *reinterpret_cast<const uint4*>(dout + off + n * R::kPass * ss) : make_uint4(0u, 0u, 0u, 0u);
    l[n] = part == 0 && i < sq ? lse[static_cast<long long>(bh) * sq + i] : INFINITY;
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const uint32_t u[4] = {x[n].x, x[n].y, x[n].z, x[n].w}, v[4] = {y[n].x, y[n].y, y[n].z, y[n].w};
    sum[n] = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sum[n] = fmaf(__uint_as_float(u[e] << 16), __uint_as_float(v[e] << 16), sum[n]);
      sum[n] = fmaf(__uint_as_float(u[e] & 0xffff0000u), __uint_as_float(v[e] & 0xffff0000u), sum[n]);
    }
  }
#pragma unroll
  for (int m = R::kLanes / 2; m > 0; m >>= 1) {
#pragma unroll
    for (int n = 0; n < 4; ++n) sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], m);
  }
  if (part == 0) {
    float* s = stats + static_cast<long long>(tile) * (2 * C::kBQ) + in_tile;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      s[n * R::kPass] = -l[n] * kLog2e;
      s[C::kBQ + n * R::kPass] = -sum[n];
    }
  }
}

// 32 columns of up to 128 rows, a row per thread, turned round so that rows are stored whole
__device__ __forceinline__ void store_rows(__nv_bfloat16* out, long long stride, int rows, const float4 (&v)[8], float mul) {
  constexpr int kPitch = 80;  // bytes: 16-byte pieces of eight rows meet in no bank
  __shared__ __align__(16) uint8_t tile[128 * kPitch];
  uint4* own = reinterpret_cast<uint4*>(tile + threadIdx.x * kPitch);
#pragma unroll
  for (int c = 0; c < 4; ++c)
    own[c] = make_uint4(pack_bf16x2(v[2 * c].x * mul, v[2 * c].y * mul), pack_bf16x2(v[2 * c].z * mul, v[2 * c].w * mul),
                        pack_bf16x2(v[2 * c + 1].x * mul, v[2 * c + 1].y * mul),
                        pack_bf16x2(v[2 * c + 1].z * mul, v[2 * c + 1].w * mul));
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int row = e * 32 + static_cast<int>(threadIdx.x) / 4, piece = threadIdx.x % 4;
    if (row < rows) reinterpret_cast<uint4*>(out + row * stride)[piece] = *reinterpret_cast<const uint4*>(tile + row * kPitch + piece * 16);
  }
}

// dq from the sums over all key tiles: scaled, rounded, in dq's layout; a block takes 32 TMEM columns of a tile.  Behind
// those blocks, dV and dK of key tiles that came in parts: the parts added in order, a block 32 columns of one of the
// two.
template <int D>
__global__ void __launch_bounds__(128) fa2_bwd_finish(const __grid_constant__ Params p, const int dq_blocks) {
  using C = Cfg<D>;
  wait_previous_kernels();
  const int row = threadIdx.x;
  int block = static_cast<int>(blockIdx.x);
  float4 v[8];
  if (block < dq_blocks) {
    const long long tile = block / (C::kDqCols / 32);
    const int c0 = block % (C::kDqCols / 32) * 32;
    const int half = static_cast<int>(tile % C::kSplit);
    const long long t = tile / C::kSplit;
    const int i = static_cast<int>(t % p.nq);
    const long long bh = t / p.nq;
    const float4* acc = reinterpret_cast<const float4*>(p.acc + tile * (C::kDqCols * 128)) + (c0 / 4) * 128 + row;
#pragma unroll
    for (int c = 0; c < 8; ++c) v[c] = __ldcs(acc + c * 128);
    const int sums = min(p.streams, contributors<D>(p, i));
    for (int q = 1; q < sums; ++q) {
      acc += p.tiles * (C::kDqCols * 128 / 4);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float4 w = __ldcs(acc + c * 128);
        v[c] = make_float4(v[c].x + w.x, v[c].y + w.y, v[c].z + w.z, v[c].w + w.w);
      }
    }
    __nv_bfloat16* out = p.dq + (bh / p.hq) * p.q_sb + (bh % p.hq) * p.q_sh + static_cast<long long>(i) * C::kBQ * p.q_ss + half * C::kDH;
    const int rows = min(C::kBQ, p.sq - i * C::kBQ);
    if constexpr (C::kTransDq) {  // a thread has a column of 32 queries
      __shared__ __align__(16) __nv_bfloat16 tile[32][128];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        tile[4 * c][row] = __float2bfloat16_rn(v[c].x * p.scale);
        tile[4 * c + 1][row] = __float2bfloat16_rn(v[c].y * p.scale);
        tile[4 * c + 2][row] = __float2bfloat16_rn(v[c].z * p.scale);
        tile[4 * c + 3][row] = __float2bfloat16_rn(v[c].w * p.scale);
      }
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int q = e * 8 + row / 16, piece = row % 16;
        if (c0 + q < rows) reinterpret_cast<uint4*>(out + (c0 + q) * p.q_ss)[piece] = reinterpret_cast<const uint4*>(tile[q])[piece];
      }
    } else {
      store_rows(out + c0, p.q_ss, rows, v, p.scale);
    }
    return;
  }
  block -= dq_blocks;
  const int c0 = block % (C::kDH / 32) * 32;
  block /= C::kDH / 32;
  const int which = block & 1;  // 0: dV, 1: dK
  block >>= 1;
  const int j = block % p.nk;
  int r = block / p.nk;
  const int parts = p.first[j + 1] - p.first[j];
  if (parts == 1) return;
  const float4* src = reinterpret_cast<const float4*>(p.partial + ((static_cast<long long>(r) * p.per_row + p.first[j]) * 2 + which) *
                                                                      (C::kDH * 128)) +
                      (c0 / 4) * 128 + row;
#pragma unroll
  for (int c = 0; c < 8; ++c) v[c] = __ldcs(src + c * 128);
  for (int q = 1; q < parts; ++q) {
    src += 2 * (C::kDH * 128) / 4;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const float4 w = __ldcs(src + c * 128);
      v[c] = make_float4(v[c].x + w.x, v[c].y + w.y, v[c].z + w.z, v[c].w + w.w);
    }
  }
  const int half = r % C::kSplit;
  r /= C::kSplit;
  __nv_bfloat16* out = (which == 0 ? p.dv : p.dk) + (r / p.hkv) * p.k_sb + (r % p.hkv) * p.k_sh +
                       static_cast<long long>(j) * kBK * p.k_ss + half * C::kDH + c0;
  store_rows(out, p.k_ss, min(kBK, p.skv - j * kBK), v, which == 0 ? 1.0f : p.scale);
}

// How a call is cut.
struct Plan {
  int part_tiles;                    // query tiles of a part (0: whole key tiles)
  int per_row;                       // units of a row
  int streams;
  uint16_t first[kMaxParted + 1];
};

// Parts cost their fp32 way through memory and pay where key tiles are few: the time of a cut, in steps, is the
// longest unit, the turns of a query tile's dQ, or the mean load of an SM with what a unit costs beside its steps (2) and what
// the ends of the SMs' queues differ by (a sixth of the longest unit, causal units being sorted by length; half of it
// otherwise), and the joining of the parts.  Whole and cut, us: B1 Hq32 Hkv8 S2048 D128 213, 136 (2 parts); B1 Hq32 Hkv4
// S1024 D128 195, 63 (8); B1 Hq16 Hkv2 S4096 D256 1290, 699 (2); where a cut does not pay, B2 Hq16 Hkv2 S4096 D256
// 1195, 1250 (2).
template <int D>
Plan plan(int batch, int hkv, int group, int nq, int nk, int causal) {
  using C = Cfg<D>;
  Plan best{};
  best.per_row = nk;
  const long long rows = static_cast<long long>(batch) * hkv * C::kSplit;
  const int sms = device_sm_count() > 0 ? device_sm_count() : 148;
  // A row's CTAs that start at once add to the same query tiles one behind the other, about 3 us each: where
  // a row's key tiles mostly start at once, dQ is gathered in several sums, as many as stay in L2 beside the rest, 72 MB.
  // With 1, 2, 3, 4 sums, us: B3 Hq12 Hkv4 1000 x 1531 D64, 9 MB a sum, 96, 76, 72, -; B1 H2 S16384 D128, 17 MB, 598, 480,
  // 451, 432; B1 Hq32 Hkv8 S2048 D128, 34 MB, 149, 144, 145, 148; B1 Hq8 Hkv2 S8192 D128, 34 MB, 494, 464, 458, 459; B1 Hq16 Hkv2
  // S4096 D256, 67 MB, 640, 642, 651, 661; B2 of it, 134 MB, 1187, 1220, 1250, 1265.
  const long long sum_bytes = std::max(1LL, rows * group * nq * (C::kDqCols * 128 * 4));
  const long long fit = (72LL << 20) / sum_bytes;
  best.streams = rows * nk > 2LL * sms ? 1 : static_cast<int>(std::max(1LL, std::min<long long>({fit, 4, nk < 4 ? nk : nk / 4})));
  if (nk > kMaxParted || rows * nk >= 8LL * sms) return best;  // enough whole tiles
  auto tiles = [&](int j) { return std::max(0, nq - (causal ? j * (kBK / C::kBQ) : 0)); };
  auto parts_of = [&](int j, int part_tiles) { return std::max(1, (tiles(j) + part_tiles - 1) / part_tiles); };
  double total = 0.0;
  for (int j = 0; j < nk; ++j) total += static_cast<double>(tiles(j)) * group * rows;
  double best_time = 0.0;
  for (int cut = 1; cut <= 16 && cut <= nq; ++cut) {
    const int part_tiles = (nq + cut - 1) / cut;
    long long units = 0, parts = 0;
    for (int j = 0; j < nk; ++j) {
      const int n = parts_of(j, part_tiles);
      units += n;
      parts += n > 1 ? n : 0;
    }
    if (units > 0xFFFF) break;
    const double longest = static_cast<double>(part_tiles) * group;
    const double joined = static_cast<double>(parts) * rows * (2.0 * C::kDH * 128 * 4) * 2.0;  // bytes written and read
    const double mean = (total + 2.0 * static_cast<double>(units) * rows) / sms;
    const double turns = 1.5 * nk / best.streams;
    const double time = std::max({longest + 2.0, turns, mean + longest / (causal ? 6 : 2)}) +
                        (parts > 0 ? (nk > 1 ? 0.5 : 1.0) + joined / 8e6 : 0.0);  // a step is about 2 us, in which 8 MB pass
    if (cut == 1 || time < 0.85 * best_time) {
      best_time = time;
      best.part_tiles = parts > 0 ? part_tiles : 0;
      best.per_row = static_cast<int>(units);
    }
  }
  if (best.part_tiles > 0) {
    int at = 0;
    for (int j = 0; j < nk; ++j) {
      best.first[j] = static_cast<uint16_t>(at);
      at += parts_of(j, best.part_tiles);
    }
    best.first[nk] = static_cast<uint16_t>(at);
  }
  return best;
}

struct Sizes {
  long long counters, stats, acc, partial, total;  // bytes
};

template <int D>
Sizes sizes(long long batch, long long hq, long long hkv, long long sq, long long skv, const Plan& plan) {
  using C = Cfg<D>;
  const long long tiles = batch * hq * ((sq + C::kBQ - 1) / C::kBQ);
  auto up = [](long long n) { return (n + 255) / 256 * 256; };
  Sizes s{};
  s.counters = up((1 + plan.streams * tiles * C::kSplit) * 4);
  s.stats = up(tiles * 2 * C::kRowBytes);
  s.acc = skv > kBK ? plan.streams * tiles * C::kSplit * C::kDqCols * 128 * 4 : 0;  // one key tile: dq is written at once
  s.partial = plan.part_tiles > 0 ? batch * hkv * C::kSplit * plan.per_row * (2LL * C::kDH * 128 * 4) : 0;
  s.total = s.counters + s.stats + s.acc + s.partial;
  return s;
}

template <int D>
Plan plan_of(int batch, int hq, int hkv, int sq, int skv, int causal) {
  return plan<D>(batch, hkv, hq / hkv, static_cast<int>((static_cast<long long>(sq) + Cfg<D>::kBQ - 1) / Cfg<D>::kBQ),
                 static_cast<int>((static_cast<long long>(skv) + kBK - 1) / kBK), causal);
}

template <int D>
int launch(const void* dout, const void* q, const void* k, const void* v, const void* o, const float* lse, void* dq,
           void* dk, void* dv, int batch, int hq, int hkv, int sq, int skv, int layout, int causal, float sm_scale,
           void* workspace, long long workspace_bytes, uint32_t* status, cudaStream_t stream) {
  using C = Cfg<D>;
  const Plan cut = plan_of<D>(batch, hq, hkv, sq, skv, causal);
  const Sizes sz = sizes<D>(batch, hq, hkv, sq, skv, cut);
  if (workspace == nullptr || workspace_bytes < sz.total || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_fa2_bwd: needs a 16-byte aligned workspace of %lld bytes", sz.total);
  // 4-D tensor maps over (d, seq, head, batch); the layout only changes the strides.
  auto make = [&](CUtensorMap* map, const void* base, int s, int h, uint32_t rows) {
    uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(s), static_cast<uint64_t>(h),
                        static_cast<uint64_t>(batch)};
    const uint64_t row = static_cast<uint64_t>(D) * 2;
    uint64_t strides[3] = {layout == TOKMIX_LAYOUT_BHSD ? row : row * h, layout == TOKMIX_LAYOUT_BHSD ? row * s : row,
                           row * s * h};
    uint32_t box[4] = {64, rows, 1, 1};
    return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  CUtensorMap mq, mdo, mk, mv;
  if (!make(&mq, q, sq, hq, C::kBQ) || !make(&mdo, dout, sq, hq, C::kBQ) || !make(&mk, k, skv, hkv, kBK) ||
      !make(&mv, v, skv, hkv, kBK))
    return TOKMIX_ERR_INVALID_ARGUMENT;

  Params p{};
  p.dq = static_cast<__nv_bfloat16*>(dq);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.dk = static_cast<__nv_bfloat16*>(dk);
  p.dv = static_cast<__nv_bfloat16*>(dv);
  const bool bhsd = layout == TOKMIX_LAYOUT_BHSD;
  p.q_sb = static_cast<long long>(D) * sq * hq;
  p.q_sh = bhsd ? static_cast<long long>(D) * sq : D;
  p.q_ss = bhsd ? D : static_cast<long long>(D) * hq;
  p.k_sb = static_cast<long long>(D) * skv * hkv;
  p.k_sh = bhsd ? static_cast<long long>(D) * skv : D;
  p.k_ss = bhsd ? D : static_cast<long long>(D) * hkv;
  p.batch = batch;
  p.hq = hq;
  p.hkv = hkv;
  p.group = hq / hkv;
  p.sq = sq;
  p.skv = skv;
  p.nq = (sq + C::kBQ - 1) / C::kBQ;
  p.nk = (skv + kBK - 1) / kBK;
  p.causal = causal ? 1 : 0;
  const long long tiles = static_cast<long long>(batch) * hq * p.nq * C::kSplit;
  if (tiles > 0xFFFFFFFll) return fail(TOKMIX_ERR_UNSUPPORTED, "tokmix_fa2_bwd: too many tiles (%lld)", tiles);
  p.scale = sm_scale;
  p.scale_log2 = sm_scale * kLog2e;
  p.status = status;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.ticket = reinterpret_cast<uint32_t*>(ws);
  p.turns = p.ticket + 1;
  p.stats = reinterpret_cast<const float*>(ws + sz.counters);
  p.acc = reinterpret_cast<float*>(ws + sz.counters + sz.stats);
  p.per_row = cut.per_row;
  p.streams = cut.streams;
  p.part_tiles = cut.part_tiles;
  p.tiles = tiles;
  if (cut.part_tiles > 0) {
    p.partial = reinterpret_cast<float*>(ws + sz.counters + sz.stats + sz.acc);
    std::copy(cut.first, cut.first + p.nk + 1, p.first);
  }
  const long long units = static_cast<long long>(batch) * hkv * C::kSplit * p.per_row;
  const long long steps = static_cast<long long>(p.nq) * p.group;
  if (units > 0x3FFFFFFFll || steps > 0x3FFFFFFFll)
    return fail(TOKMIX_ERR_UNSUPPORTED, "tokmix_fa2_bwd: too many tiles (%lld x %lld)", units, steps);
  p.units = static_cast<int>(units);
  // The rows of a wave fill the SMs with this many key tiles each: fewer wait less for each other's turns, more read the same
  // queries together.  Several heads give the turns time, and a causal row's tiles are of different length (us, B4 Hq32 Hkv8
  // S8192 D128 causal: 6842 at 4, 6623 at 8, 6779 at 16; D64 4235 at 4, 4115 at 8; B8 H8 S2048 causal D64: 171 at 1 and 2, 184
  // at 4, 200 at 6; D128 280, 283, 294).  Without a mask the units are of one length, and those that start at once should be the
  // same number of key tiles in every row: B16 H12 S512 D64, 192 rows, 86 at 2, 102 at 4; B4 H16 S2048 D128, 64 rows, 486 at
  // 2 (2.3 a row), 445 at 4, 453 at 6.
  const int sms = std::max(1, device_sm_count());
  const long long kv_rows = static_cast<long long>(batch) * hkv * C::kSplit;
  const int share = p.group > 1 ? 8 : causal || kv_rows >= (sms + 1) / 2 ? 2 : 4;
  p.wave = (sms + share - 1) / share;

  const long long blocks = static_cast<long long>(batch) * hq * p.nq * Prep<D>::kBlocks;
  if (blocks > 0x7FFFFFFFll) return fail(TOKMIX_ERR_UNSUPPORTED, "tokmix_fa2_bwd: too many query tiles (%lld)", blocks);
  const int smem_bytes = C::kBytes;
  if (!ensure_smem_attr(reinterpret_cast<const void*>(&fa2_bwd_kernel<D>), smem_bytes))
    return check_launch("tokmix_fa2_bwd: cudaFuncSetAttribute");
  cudaError_t e = launch_overlapped(&fa2_bwd_prep<D>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream,
                                    static_cast<const __nv_bfloat16*>(o), static_cast<const __nv_bfloat16*>(dout), lse,
                                    const_cast<float*>(p.stats), p.ticket, sz.counters / 4, sq, p.nq, hq,
                                    p.q_sb, p.q_sh, p.q_ss);
  if (e == cudaSuccess) {
    const int grid = static_cast<int>(std::min<long long>(units, std::max(1, device_sm_count())));
    e = launch_overlapped(&fa2_bwd_kernel<D>, dim3(static_cast<unsigned>(grid)), dim3(Cfg<D>::kThreads),
                          static_cast<size_t>(smem_bytes), stream, mq, mdo, mk, mv, p);
  }
  const long long dq_blocks = p.nk > 1 ? tiles * (C::kDqCols / 32) : 0;
  const long long join_blocks = cut.part_tiles > 0 ? static_cast<long long>(batch) * hkv * C::kSplit * p.nk * 2 * (C::kDH / 32) : 0;
  if (e == cudaSuccess && dq_blocks + join_blocks > 0)
    e = launch_overlapped(&fa2_bwd_finish<D>, dim3(static_cast<unsigned>(dq_blocks + join_blocks)), dim3(128), 0, stream, p,
                          static_cast<int>(dq_blocks));
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(TOKMIX_ERR_LAUNCH, "tokmix_fa2_bwd: %s", cudaGetErrorString(e));
  }
  return check_launch("tokmix_fa2_bwd");
}

// The function for a head_dim, or `otherwise` where there is no kernel for it
template <typename F64, typename F128, typename F256>
auto by_head_dim(int head_dim, F64 f64, F128 f128, F256 f256, decltype(f64()) otherwise) {
  return head_dim == 64 ? f64() : head_dim == 128 ? f128() : head_dim == 256 ? f256() : otherwise;
}

}  // namespace fa2b
}  // namespace tokmix

extern "C" long long tokmix_fa2_bwd_workspace_bytes(int batch, int heads_q, int heads_kv, int seqlen_q, int seqlen_kv,
                                                    int head_dim, int causal) {
  using namespace tokmix::fa2b;
  if (batch < 0 || heads_q <= 0 || heads_kv <= 0 || heads_q % heads_kv != 0 || seqlen_q < 0 || seqlen_kv < 0) return -1;
  auto need = [&](auto d) {
    constexpr int D = decltype(d)::value;
    return sizes<D>(batch, heads_q, heads_kv, seqlen_q, seqlen_kv, plan_of<D>(batch, heads_q, heads_kv, seqlen_q, seqlen_kv, causal))
        .total;
  };
  return by_head_dim(
      head_dim, [&] { return need(std::integral_constant<int, 64>()); }, [&] { return need(std::integral_constant<int, 128>()); },
      [&] { return need(std::integral_constant<int, 256>()); }, -1LL);
}

extern "C" int tokmix_fa2_bwd(const void* dout, const void* q, const void* k, const void* v, const void* o,
                              const float* lse, void* dq, void* dk, void* dv, int batch, int heads_q, int heads_kv,
                              int seqlen_q, int seqlen_kv, int head_dim, int layout, int causal, float sm_scale,
                              void* workspace, long long workspace_bytes, uint32_t* status, void* stream) {
  using namespace tokmix;
  if (batch < 0 || heads_q <= 0 || heads_kv <= 0 || seqlen_q < 0 || seqlen_kv < 0)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_fa2_bwd: negative or zero size");
  if (heads_q % heads_kv != 0)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_fa2_bwd: heads_q (%d) must be a multiple of heads_kv (%d)", heads_q,
                heads_kv);
  if (layout != TOKMIX_LAYOUT_BHSD && layout != TOKMIX_LAYOUT_BSHD)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_fa2_bwd: unknown layout %d", layout);
  if (!(sm_scale > 0.0f) || !std::isfinite(sm_scale))
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_fa2_bwd: sm_scale must be finite and positive");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(TOKMIX_ERR_UNSUPPORTED, "tokmix_fa2_bwd: head_dim %d not supported (64, 128 or 256)", head_dim);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (batch == 0 || (seqlen_q == 0 && seqlen_kv == 0)) return TOKMIX_OK;
  if (std::max(seqlen_q, seqlen_kv) > 0x7FFFFFFF - (fa2b::kBK - 1))  // whole tiles are counted in int
    return fail(TOKMIX_ERR_UNSUPPORTED, "tokmix_fa2_bwd: too many tokens (%d, %d)", seqlen_q, seqlen_kv);
  if (seqlen_kv == 0)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_fa2_bwd: seqlen_kv must be positive when seqlen_q is");
  for (const void* ptr : {k, v, static_cast<const void*>(dk), static_cast<const void*>(dv)})
    if (ptr == nullptr || reinterpret_cast<uintptr_t>(ptr) % 16 != 0)
      return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_fa2_bwd: tensors must be non-null and 16-byte aligned");
  if (seqlen_q > 0) {
    for (const void* ptr : {dout, q, o, static_cast<const void*>(dq)})
      if (ptr == nullptr || reinterpret_cast<uintptr_t>(ptr) % 16 != 0)
        return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_fa2_bwd: tensors must be non-null and 16-byte aligned");
    if (lse == nullptr) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_fa2_bwd: null lse");
  }
  if (const int rc = check_device()) return rc;
  if (seqlen_q == 0) {  // no query: no gradient reaches the keys and values
    const size_t bytes = static_cast<size_t>(batch) * heads_kv * seqlen_kv * head_dim * 2;
    if (cudaMemsetAsync(dk, 0, bytes, s) != cudaSuccess || cudaMemsetAsync(dv, 0, bytes, s) != cudaSuccess)
      return check_launch("tokmix_fa2_bwd");
    return TOKMIX_OK;
  }
  auto run = [&](auto d) {
    return fa2b::launch<decltype(d)::value>(dout, q, k, v, o, lse, dq, dk, dv, batch, heads_q, heads_kv, seqlen_q,
                                            seqlen_kv, layout, causal, sm_scale, workspace, workspace_bytes, status, s);
  };
  return fa2b::by_head_dim(
      head_dim, [&] { return run(std::integral_constant<int, 64>()); }, [&] { return run(std::integral_constant<int, 128>()); },
      [&] { return run(std::integral_constant<int, 256>()); }, static_cast<int>(TOKMIX_ERR_UNSUPPORTED));
}
