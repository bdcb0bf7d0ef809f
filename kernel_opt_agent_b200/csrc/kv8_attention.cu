// kv8_attention.cu -- attention of a few new tokens per sequence over the paged 8-bit cache.
//
// Maths, per query row r (a new token and a query head) over the cached tokens j it sees:
//   s_j = sm_scale (q . k8_j) ks_j,   o = sum_j e^{s_j} vs_j v8_j / sum_j e^{s_j}
// with k8, v8 the cached bytes' values and ks, vs the scales of token j's (page, head).
//
// Bound: HBM, the cache's bytes (4 heads_q / heads_kv flops per byte).  So the rows that read the same keys
// and values -- the tokens and heads of a group -- share one pass over them, and the work is cut along the
// sequences so that every SM streams until the end:
//   * a unit is (sequence, key/value head, tile of 8 or 16 rows); its tokens come in tiles of 4 KB of keys and
//     4 KB of values (16, 32 or 64 tokens).  All units' tiles laid end to end are cut into equal ranges, one
//     per CTA of a grid that fills the GPU once; lengths are read on the device, so the launch does not depend
//     on them.  A unit inside one range is written directly; a unit cut by range borders leaves normalised
//     partial rows with their maximum and sum, and a second kernel joins them in the order of the CTAs
//     (launched to start as the first drains; results do not depend on timing).
//   * a warp takes every fourth tile of its CTA's range, loads it straight into registers with 16-byte loads
//     (the order of the head dimension inside a product is free, so a lane's 16 bytes are its fragments), and
//     loads the next tile's keys as soon as this tile's scores stand and its values as soon as they are
//     used up: 8 KB in flight per warp, 12 warps per SM.  No shared memory, barrier or wait is on that path.
//   * scores S^T = K Q^T and outputs O^T = V^T P^T are m16n8k16 products with the cache's bytes as the 16-row
//     operand: e4m3 and int8 values are exact in fp16, accumulation is fp32.  The tensor core's newer path
//     (tcgen05) would want the bytes in shared memory and 128-row tiles of them for 8 to 16 query rows; the
//     products take a tenth of the time the bytes do, so registers are the shorter way.
//
// Number formats.  q rows enter fp16 after scaling by a power of two that brings their largest element to
// [2^14, 2^15): exact for elements down to 2^-28 of it (bf16 has 8 bits, fp16 11).  Weights enter as
// 2^14 e^{s_j - m} rounded to fp16 (half a step is 2^-11; under 2^-38 of the largest they vanish), times
// vs_j / vref, vref the largest value scale a warp has met -- powers of two, so exact; a block whose scale is under
// 2^-28 of vref loses bits that are 2^-39 of the largest block's values.  Maxima, sums and outputs are fp32.
#include "kv8_common.cuh"

#include <algorithm>
#include <cmath>

namespace tokmix {
namespace kv8 {

constexpr int kMaxTokens = 16;
constexpr int kMaxBatch = 8192;  // the plan keeps batch + 1 words in shared memory
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kShift = 14.0f;  // weights are held times 2^14
constexpr int kJoinThreads = 256;
constexpr int kMaxCtas = 148 * 8;

template <int D, int NT>
struct Shape {
  static constexpr int kTok = 4096 / D;       // tokens per tile
  static constexpr int kMt = kTok / 16;       // 16-token subtiles (a page holds whole ones)
  static constexpr int kRows = 8 * NT;        // query rows per unit
  static constexpr int kQStride = D + 8;      // halves between rows of q in shared memory (conflict-free 16-byte reads)
  static constexpr int kCtasPerSm = NT == 1 ? 3 : 2;
  static constexpr int kMergeBytes = kWarps * kRows * D * 4;
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
  uint32_t* status;
};

// ------------------------------------------------------------------------------------ the plan
struct Unit {
  int tiles;      // token tiles of each of the sequence's units
  int row_tiles;  // row tiles per key/value head
};

template <int TOK, int ROWS>
__device__ __forceinline__ Unit unit_of(const AttnParams& p, const Seq& s) {
  Unit u;
  u.tiles = (s.end + TOK - 1) / TOK;
  u.row_tiles = ((s.end - s.start) * p.group + ROWS - 1) / ROWS;
  return u;
}

// prefix[b] = tiles of the sequences before b (exclusive), prefix[batch] = all; every thread calls.
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
      n = static_cast<uint32_t>(u.tiles) * u.row_tiles * p.c.hkv;
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

// CTAs that take part: each has at least a tile per warp, so none is empty
__device__ __forceinline__ uint32_t active_ctas(const AttnParams& p, uint32_t total) {
  return min(static_cast<uint32_t>(p.grid), max(1u, total / kWarps));
}
__device__ __forceinline__ uint32_t range_begin(uint32_t cta, uint32_t total, uint32_t ctas) {
  return static_cast<uint32_t>(static_cast<unsigned long long>(cta) * total / ctas);
}
// the CTA whose range holds tile t: the last one with range_begin <= t
__device__ __forceinline__ uint32_t cta_of(uint32_t t, uint32_t total, uint32_t ctas) {
  return static_cast<uint32_t>(((static_cast<unsigned long long>(t) + 1) * ctas - 1) / total);
}

// ------------------------------------------------------------------------------------ small pieces
__device__ __forceinline__ uint4 ld16(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld8(const uint8_t* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

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

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float nan_f() { return __uint_as_float(0x7fc00000u); }

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
template <int D, bool E4M3, int NT>
__global__ void __launch_bounds__(kThreads, Shape<D, NT>::kCtasPerSm) attn_kernel(const AttnParams p) {
  using S = Shape<D, NT>;
  constexpr int TOK = S::kTok, MT = S::kMt, ROWS = S::kRows, J = D / 64;
  constexpr int kVec = D / 8;  // 16-byte vectors of a query row
  extern __shared__ __align__(16) uint8_t smem[];
  float* merge = reinterpret_cast<float*>(smem);                                   // [warp][row][D]
  __half* qs = reinterpret_cast<__half*>(smem + S::kMergeBytes);                    // [row][kQStride]
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem + S::kMergeBytes + ROWS * S::kQStride * 2);
  __shared__ float row_factor[ROWS], warp_m[kWarps][ROWS], warp_l[kWarps][ROWS], warp_v[kWarps];
  __shared__ uint32_t scratch[kWarps];

  const View& c = p.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, cq = lane & 3;

  asm volatile("griddepcontrol.launch_dependents;");
  make_plan<TOK, ROWS, kThreads>(p, prefix, scratch);
  const uint32_t total = prefix[c.batch];
  if (total == 0) return;
  const uint32_t ctas = active_ctas(p, total);
  if (blockIdx.x >= ctas) return;
  uint32_t pos = range_begin(blockIdx.x, total, ctas);
  const uint32_t stop = range_begin(blockIdx.x + 1, total, ctas);
  int b = 0;
  for (int hi = c.batch; hi - b > 1;) {  // the last b with prefix[b] <= pos
    const int mid = (b + hi) >> 1;
    if (prefix[mid] <= pos) b = mid; else hi = mid;
  }

  for (bool first = true; pos < stop; first = false) {
    while (prefix[b + 1] <= pos) ++b;
    const Seq s = load_seq(c, b, p.tokens);
    const Unit u = unit_of<TOK, ROWS>(p, s);
    const int off = static_cast<int>(pos - prefix[b]);
    const int ui = off / u.tiles;
    const int t0 = off - ui * u.tiles;
    const int t1 = min(u.tiles, t0 + static_cast<int>(stop - pos));
    const int kvh = ui / u.row_tiles;
    const int row0 = (ui - kvh * u.row_tiles) * ROWS;     // first row of the unit
    const int rows_valid = (s.end - s.start) * p.group;   // rows of the sequence's key/value head
    pos += t1 - t0;

    // q rows into shared memory as scaled halves; rows behind the last are zero and never written out
    for (int v = threadIdx.x; v < ROWS * kVec; v += kThreads) {
      const int r = v / kVec, x = v % kVec;
      const int row = row0 + r;
      float f[8];
      float amax = 0.0f;
      if (row < rows_valid) {
        const int i = row / p.group, h = kvh * p.group + row - i * p.group;
        const long long at = b * p.q_sb + i * p.q_st + h * p.q_sh + x * 8;
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + at));
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 t = p.bf16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&ws[e]))
                                  : __half22float2(*reinterpret_cast<const __half2*>(&ws[e]));
          f[2 * e] = t.x;
          f[2 * e + 1] = t.y;
          amax = fmaxf(amax, fmaxf(fabsf(t.x), fabsf(t.y)));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 0.0f;
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
      *reinterpret_cast<uint4*>(qs + r * S::kQStride + x * 8) = hq;
    }
    __syncthreads();

    // this lane's rows (columns of the products): 8 nt + 2 cq + {0, 1}
    float factor[NT][2], m[NT][2], l[NT][2];
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
        m[nt][e] = -INFINITY;
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
    float vref = 0.0f;

    const int32_t* trow = c.table + static_cast<long long>(b) * c.table_stride;
    const uint8_t* kbase = c.k + kvh * c.k_head_stride + g * D + 16 * cq;
    const uint8_t* vbase = c.v + kvh * c.v_head_stride + 2 * cq * D + (D == 64 ? 8 : 16) * g;
    const float* ksb = c.k_scale + kvh;
    const float* vsb = c.v_scale + kvh;

    uint4 kr[8];
    uint32_t vr[32];
    int pid[MT];
    float ks[MT], vs[MT], ksn[MT], vsn[MT];

    // page of each 16-token subtile of tile t; -1: outside the pool, -2: behind the range or the sequence
    auto load_pages = [&](int t) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int tok = t * TOK + mt * 16;
        pid[mt] = -2;
        if (t < t1 && tok < s.end) {
          pid[mt] = __ldg(trow + (tok >> c.page_shift));
          if (static_cast<unsigned>(pid[mt]) >= static_cast<unsigned>(c.num_pages)) {
            pid[mt] = -1;
            if (lane == 0) report_bad(p.status);
          }
        }
      }
    };
    auto load_keys = [&](int t) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if (pid[mt] >= 0) {
          const int slot = (t * TOK + mt * 16) & (c.page - 1);
          const uint8_t* src = kbase + pid[mt] * c.k_page_stride + slot * D;
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int j = 0; j < J; ++j) kr[(mt * 2 + half) * J + j] = ld16(src + half * 8 * D + j * 64);
          ksn[mt] = __ldg(ksb + static_cast<long long>(pid[mt]) * c.hkv);
          vsn[mt] = __ldg(vsb + static_cast<long long>(pid[mt]) * c.hkv);
        } else {
#pragma unroll
          for (int x = 0; x < 2 * J; ++x) kr[mt * 2 * J + x] = make_uint4(0u, 0u, 0u, 0u);
          ksn[mt] = pid[mt] == -1 ? nan_f() : 0.0f;  // NaN scores for the rows that see it
          vsn[mt] = 0.0f;
        }
      }
    };
    // vr[(mt * 4 + i) * (D / 32) + ...]: token 2 cq + {0, 1, 8, 9}[i] of subtile mt, this lane's D / 8 dims
    auto load_values = [&](int t) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if (pid[mt] >= 0) {
          const int slot = (t * TOK + mt * 16) & (c.page - 1);
          const uint8_t* src = vbase + pid[mt] * c.v_page_stride + slot * D;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint8_t* tp = src + ((i & 1) + (i >> 1) * 8) * D;
            if constexpr (D == 64) {
              const uint2 v = ld8(tp);
              vr[(mt * 4 + i) * 2] = v.x;
              vr[(mt * 4 + i) * 2 + 1] = v.y;
            } else {
#pragma unroll
              for (int jj = 0; jj < D / 128; ++jj) {
                const uint4 v = ld16(tp + jj * 128);
                uint32_t* d = vr + (mt * 4 + i) * (D / 32) + jj * 4;
                d[0] = v.x;
                d[1] = v.y;
                d[2] = v.z;
                d[3] = v.w;
              }
            }
          }
        } else {
#pragma unroll
          for (int x = 0; x < D / 8; ++x) vr[mt * (D / 8) + x] = 0u;
        }
      }
    };

    int t = t0 + warp;
    load_pages(t);
    load_keys(t);
    load_values(t);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      ks[mt] = ksn[mt];
      vs[mt] = vsn[mt];
    }
    load_pages(t + kWarps);

    for (; t < t1; t += kWarps) {
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
          const uint4 lo = kr[mt * 2 * J + j], hi = kr[(mt * 2 + 1) * J + j];
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
      load_keys(t + kWarps);

      // softmax: a lane has tokens g and g + 8 of each subtile for its rows
      float top[NT][2];
      const bool tail = t * TOK + TOK > min_lim;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[nt][e] = -INFINITY;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float& x = sc[mt][nt][0][half * 2 + e];
              x = (x + sc[mt][nt][1][half * 2 + e]) * (ks[mt] * factor[nt][e]);
              if (tail && t * TOK + mt * 16 + half * 8 + g >= lim[nt][e]) x = -INFINITY;
              top[nt][e] = fmaxf(top[nt][e], x);
            }
          }
        }
      }
      bool grew = false;
      float ref[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) top[nt][e] = fmaxf(top[nt][e], __shfl_xor_sync(0xffffffffu, top[nt][e], o));
          top[nt][e] = fmaxf(top[nt][e], m[nt][e]);
          grew |= top[nt][e] > m[nt][e];
          ref[nt][e] = top[nt][e] == -INFINITY ? 0.0f : top[nt][e];  // a row that has seen nothing yet
        }
      }
      float vnew = vref;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) vnew = fmaxf(vnew, vs[mt]);
      if (__any_sync(0xffffffffu, grew) || vnew > vref) {
        const float vcorr = vnew > vref ? vref / vnew : 1.0f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float c0 = ex2(m[nt][0] - ref[nt][0]), c1 = ex2(m[nt][1] - ref[nt][1]);
          l[nt][0] *= c0;
          l[nt][1] *= c1;
          m[nt][0] = top[nt][0];
          m[nt][1] = top[nt][1];
          const float a0 = c0 * vcorr, a1 = c1 * vcorr;
#pragma unroll
          for (int x = 0; x < D / 16; ++x) {
            acc[nt][x][0] *= a0;
            acc[nt][x][1] *= a1;
            acc[nt][x][2] *= a0;
            acc[nt][x][3] *= a1;
          }
        }
        vref = vnew;
      }
      uint32_t pb[MT][NT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const float rv = vref > 0.0f ? vs[mt] / vref : vs[mt] * 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float w0 = ex2(sc[mt][nt][0][half * 2] - (ref[nt][0] - kShift));
            const float w1 = ex2(sc[mt][nt][0][half * 2 + 1] - (ref[nt][1] - kShift));
            l[nt][0] += w0;
            l[nt][1] += w1;
            // a hidden token weighs nothing even where its block's scale is NaN
            const float p0 = sc[mt][nt][0][half * 2] == -INFINITY ? 0.0f : w0 * rv;
            const float p1 = sc[mt][nt][0][half * 2 + 1] == -INFINITY ? 0.0f : w1 * rv;
            pb[mt][nt][half] = transpose8x8(half2_bits(p0, p1));
          }
        }
      }
      // bytes behind the sequence's end may be anything, e4m3 NaN too, and 0 * NaN would stay
      if (t * TOK + TOK > s.end) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (t * TOK + mt * 16 + 2 * cq + (i & 1) + (i >> 1) * 8 >= s.end) {
#pragma unroll
              for (int x = 0; x < D / 32; ++x) vr[(mt * 4 + i) * (D / 32) + x] = 0u;
            }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          const uint32_t* w = vr + mt * (D / 8) + x;  // four dims of tokens 2cq, +1, +8, +9
          const uint32_t t0w = w[0], t1w = w[D / 32], t8w = w[2 * (D / 32)], t9w = w[3 * (D / 32)];
#pragma unroll
          for (int y = 0; y < 2; ++y) {  // dims 4x + 2y, 4x + 2y + 1
            uint32_t a0, a1, a2, a3;
            widen4<E4M3>(__byte_perm(t0w, t1w, y == 0 ? 0x5140 : 0x7362), a0, a1);
            widen4<E4M3>(__byte_perm(t8w, t9w, y == 0 ? 0x5140 : 0x7362), a2, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(acc[nt][2 * x + y], a0, a1, a2, a3, pb[mt][nt][0], pb[mt][nt][1]);
          }
        }
      }
      load_values(t + kWarps);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        ks[mt] = ksn[mt];
        vs[mt] = vsn[mt];
      }
      load_pages(t + 2 * kWarps);
    }

    // join the four warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], o);
        const int r = nt * 8 + 2 * cq + e;
        if (g == 0) {
          warp_m[warp][r] = m[nt][e];
          warp_l[warp][r] = l[nt][e];
        }
        // dims of acc[2x], acc[2x + 1]: D 64: 8 g + 4 x; else 128 (x / 4) + 16 g + 4 (x % 4), four in a row
        float* dst = merge + (warp * ROWS + r) * D + (D == 64 ? 8 : 16) * g;
#pragma unroll
        for (int x = 0; x < D / 32; ++x)
          *reinterpret_cast<float4*>(dst + (D == 64 ? 4 * x : 128 * (x / 4) + 4 * (x % 4))) =
              make_float4(acc[nt][2 * x][e], acc[nt][2 * x][2 + e], acc[nt][2 * x + 1][e], acc[nt][2 * x + 1][2 + e]);
      }
    }
    if (lane == 0) warp_v[warp] = vref;
    __syncthreads();
    const bool whole = t0 == 0 && t1 == u.tiles;
    const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (first ? 0 : 1);
    for (int v = threadIdx.x; v < ROWS * (D / 4); v += kThreads) {
      const int r = v / (D / 4), x = v % (D / 4);
      const int row = row0 + r;
      if (row >= rows_valid) continue;
      float top = -INFINITY, sum = 0.0f, w[kWarps];
#pragma unroll
      for (int i = 0; i < kWarps; ++i) top = fmaxf(top, warp_m[i][r]);
      const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        w[i] = ex2(warp_m[i][r] - ref);
        sum += w[i] * warp_l[i][r];
      }
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const float4 a = *reinterpret_cast<const float4*>(merge + (i * ROWS + r) * D + 4 * x);
        const float wi = w[i] * inv, vi = warp_v[i];
        o[0] += a.x * wi * vi;
        o[1] += a.y * wi * vi;
        o[2] += a.z * wi * vi;
        o[3] += a.w * wi * vi;
      }
      if (whole) {
        const int i = row / p.group, h = kvh * p.group + row - i * p.group;
        const size_t orow = (static_cast<size_t>(b) * p.tokens + i) * p.hq + h;
        store_out4(p, orow * D + 4 * x, o);
        if (p.lse != nullptr && x == 0) p.lse[orow] = lse_of(ref, sum);
      } else {
        *reinterpret_cast<float4*>(p.part_o + (slot * ROWS + r) * D + 4 * x) = make_float4(o[0], o[1], o[2], o[3]);
        if (x == 0) p.part_ml[slot * ROWS + r] = make_float2(top, sum);
      }
    }
    __syncthreads();  // before the next segment's q and sums
  }
}

// ------------------------------------------------------------------------------------ joining cut units
// Rows of units that range borders cut (partials of CTAs c0 .. c1), rows that see nothing (zeros) and rows of
// sequences whose lengths do not fit (NaN).  A CTA takes up to 8 rows, a warp each; a row with many partials is
// joined by the whole CTA.
template <int D, int NT>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const AttnParams p, int rows_per_cta) {
  using S = Shape<D, NT>;
  constexpr int TOK = S::kTok, ROWS = S::kRows, kShort = 8;
  constexpr int TPR = D / 4, PG = kJoinThreads / TPR;  // threads of a partial row, partials at a time
  extern __shared__ __align__(16) uint8_t smem[];
  float* weight = reinterpret_cast<float*>(smem);                       // [kMaxCtas]
  float4* sums = reinterpret_cast<float4*>(smem + kMaxCtas * 4);        // [PG][TPR]
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem + kMaxCtas * 4 + kJoinThreads * 16);
  __shared__ uint32_t scratch[kJoinThreads / 32];
  __shared__ float red[2][kJoinThreads / 32];
  __shared__ uint32_t long_c0[8], long_c1[8], long_t0[8];
  __shared__ int long_r[8];
  __shared__ long long long_row[8];

  make_plan<TOK, ROWS, kJoinThreads>(p, prefix, scratch);  // reads only the call's inputs
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t total = prefix[p.c.batch];
  const uint32_t ctas = active_ctas(p, total);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long rows = static_cast<long long>(p.c.batch) * p.tokens * p.hq;
  const long long step = static_cast<long long>(gridDim.x) * rows_per_cta;
  for (long long base = static_cast<long long>(blockIdx.x) * rows_per_cta; base < rows; base += step) {
    const long long row = base + warp;
    if (lane == 0) long_c1[warp] = 0;
    if (warp < rows_per_cta && row < rows) {
      const int h = static_cast<int>(row % p.hq);
      const int rest = static_cast<int>(row / p.hq);
      const int i = rest % p.tokens, b = rest / p.tokens;
      const Seq s = load_seq(p.c, b, p.tokens);
      if (!s.ok || i >= s.end - s.start) {
        const float f = s.ok ? 0.0f : nan_f();
        const float o[4] = {f, f, f, f};
        for (int x = lane; x < TPR; x += 32) store_out4(p, static_cast<size_t>(row) * D + 4 * x, o);
        if (p.lse != nullptr && lane == 0) p.lse[row] = s.ok ? -INFINITY : nan_f();
      } else {
        const Unit u = unit_of<TOK, ROWS>(p, s);
        const int kvh = h / p.group, r = i * p.group + h - kvh * p.group;
        const uint32_t first = prefix[b] + static_cast<uint32_t>(kvh * u.row_tiles + r / ROWS) * u.tiles;
        const uint32_t c0 = cta_of(first, total, ctas), c1 = cta_of(first + u.tiles - 1, total, ctas);
        const int rr = r % ROWS;
        if (c1 - c0 >= kShort) {
          if (lane == 0) {
            long_c0[warp] = c0;
            long_c1[warp] = c1;
            long_t0[warp] = first;
            long_r[warp] = rr;
            long_row[warp] = row;
          }
        } else if (c1 > c0) {
          // the partial of CTA c: its first segment unless the unit began inside its range
          const uint32_t c = c0 + min(static_cast<uint32_t>(lane), c1 - c0);
          const size_t slot = 2 * static_cast<size_t>(c) + (range_begin(c, total, ctas) >= first ? 0 : 1);
          const float2 ml = lane <= static_cast<int>(c1 - c0) ? p.part_ml[slot * ROWS + rr] : make_float2(-INFINITY, 0.0f);
          float top = ml.x;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const float ref = top == -INFINITY ? 0.0f : top;
          const float w = ex2(ml.x - ref) * ml.y;
          float sum = w;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          constexpr int X = (TPR + 31) / 32;
          float acc[X][4];
#pragma unroll
          for (int x = 0; x < X; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[x][e] = 0.0f;
#pragma unroll
          for (int k = 0; k < kShort; ++k) {
            if (k > static_cast<int>(c1 - c0)) break;
            const float wk = __shfl_sync(0xffffffffu, w, k) * inv;
            const size_t sk = 2 * static_cast<size_t>(c0 + k) + (range_begin(c0 + k, total, ctas) >= first ? 0 : 1);
            const float4* src = reinterpret_cast<const float4*>(p.part_o + (sk * ROWS + rr) * D);
#pragma unroll
            for (int x = 0; x < X; ++x) {
              if (lane + 32 * x < TPR) {
                const float4 a = __ldcg(src + lane + 32 * x);
                acc[x][0] += wk * a.x;
                acc[x][1] += wk * a.y;
                acc[x][2] += wk * a.z;
                acc[x][3] += wk * a.w;
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
      const int n = static_cast<int>(c1 - c0) + 1, rr = long_r[k];
      const uint32_t first = long_t0[k];
      float top = -INFINITY;
      for (int x = threadIdx.x; x < n; x += kJoinThreads) {
        const size_t slot = 2 * static_cast<size_t>(c0 + x) + (range_begin(c0 + x, total, ctas) >= first ? 0 : 1);
        top = fmaxf(top, __ldcg(&p.part_ml[slot * ROWS + rr]).x);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (lane == 0) red[0][warp] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kJoinThreads / 32; ++w) top = fmaxf(top, red[0][w]);
      const float ref = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f;
      for (int x = threadIdx.x; x < n; x += kJoinThreads) {
        const size_t slot = 2 * static_cast<size_t>(c0 + x) + (range_begin(c0 + x, total, ctas) >= first ? 0 : 1);
        const float2 ml = __ldcg(&p.part_ml[slot * ROWS + rr]);
        const float w = ex2(ml.x - ref) * ml.y;
        weight[x] = w;
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
      const int x = threadIdx.x % TPR, pg = threadIdx.x / TPR;
      float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
      for (int y = pg; y < n; y += PG) {
        const size_t slot = 2 * static_cast<size_t>(c0 + y) + (range_begin(c0 + y, total, ctas) >= first ? 0 : 1);
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part_o + (slot * ROWS + rr) * D) + x);
        const float w = weight[y] * inv;
        a.x += w * v.x;
        a.y += w * v.y;
        a.z += w * v.z;
        a.w += w * v.w;
      }
      sums[pg * TPR + x] = a;
      __syncthreads();
      if (pg == 0) {
        float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int y = 0; y < PG; ++y) {
          const float4 v = sums[y * TPR + x];
          o[0] += v.x;
          o[1] += v.y;
          o[2] += v.z;
          o[3] += v.w;
        }
        store_out4(p, static_cast<size_t>(long_row[k]) * D + 4 * x, o);
        if (p.lse != nullptr && x == 0) p.lse[long_row[k]] = lse_of(ref, sum);
      }
      __syncthreads();  // before the next row's weights and sums
    }
    __syncthreads();  // before the next rows' descriptions
  }
}

template <int D, int NT>
size_t workspace_bytes(int sms) {
  using S = Shape<D, NT>;
  const size_t slots = 2 * static_cast<size_t>(sms) * S::kCtasPerSm;
  return slots * S::kRows * (D * 4 + 8);
}

template <int D, bool E4M3, int NT>
int launch_attn(const char* who, AttnParams& p, int sms, void* workspace, cudaStream_t s) {
  using S = Shape<D, NT>;
  p.grid = sms * S::kCtasPerSm;
  if (p.grid > kMaxCtas) return fail(TOKMIX_ERR_UNSUPPORTED, "%s: more SMs than the kernel is planned for", who);
  const size_t slots = 2 * static_cast<size_t>(p.grid);
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + slots * S::kRows * D);
  const int plan = (p.c.batch + 1) * 4;
  const int smem = S::kMergeBytes + S::kRows * S::kQStride * 2 + plan;
  const int join_smem = kMaxCtas * 4 + kJoinThreads * 16 + plan;
  // limits for the largest batch, set once
  const int plan_max = (kMaxBatch + 1) * 4;
  auto* attn = attn_kernel<D, E4M3, NT>;
  auto* join = join_kernel<D, NT>;
  if (!ensure_smem_attr(reinterpret_cast<const void*>(attn), S::kMergeBytes + S::kRows * S::kQStride * 2 + plan_max) ||
      !ensure_smem_attr(reinterpret_cast<const void*>(join), kMaxCtas * 4 + kJoinThreads * 16 + plan_max))
    return fail(TOKMIX_ERR_LAUNCH, "%s: cannot set the shared memory size", who);
  attn<<<p.grid, kThreads, smem, s>>>(p);
  if (const int rc = check_launch(who)) return rc;
  const long long rows = static_cast<long long>(p.c.batch) * p.tokens * p.hq;
  const int per = static_cast<int>(std::min<long long>(8, (rows + 2 * sms - 1) / (2 * sms)));
  const long long want = (rows + per - 1) / per;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<long long>(want, 4LL * sms)));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(join_smem);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, join, static_cast<const AttnParams>(p), per) != cudaSuccess) return check_launch(who);
  return check_launch(who);
}

template <int D>
int dispatch_attn(const char* who, AttnParams& p, bool e4m3, int sms, void* ws, cudaStream_t s) {
  // up to 8 query rows share a pass (8 columns of the product), else 16
  if (p.tokens * p.group <= 8)
    return e4m3 ? launch_attn<D, true, 1>(who, p, sms, ws, s) : launch_attn<D, false, 1>(who, p, sms, ws, s);
  return e4m3 ? launch_attn<D, true, 2>(who, p, sms, ws, s) : launch_attn<D, false, 2>(who, p, sms, ws, s);
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
  const bool one = static_cast<long long>(tokens) * (heads_q / heads_kv) <= 8;
  size_t n = 0;
  if (head_dim == 64)
    n = one ? workspace_bytes<64, 1>(sms) : workspace_bytes<64, 2>(sms);
  else if (head_dim == 128)
    n = one ? workspace_bytes<128, 1>(sms) : workspace_bytes<128, 2>(sms);
  else
    n = one ? workspace_bytes<256, 1>(sms) : workspace_bytes<256, 2>(sms);
  return static_cast<long long>(n);
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
  if (!q || !out || !workspace) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: null pointer argument", who);
  if (reinterpret_cast<uintptr_t>(q) % 16 != 0 || reinterpret_cast<uintptr_t>(out) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: tensors must be 16-byte aligned", who);
  for (const long long st : {q_batch_stride, q_token_stride, q_head_stride})
    if (st % 8 != 0 || st < 0)
      return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: strides of q must be multiples of 8 elements", who);
  if (p.c.batch > kMaxBatch) return fail(TOKMIX_ERR_UNSUPPORTED, "%s: at most %d sequences (got %d)", who, kMaxBatch, p.c.batch);
  const long long most_tiles = (static_cast<long long>(p.c.max_pages) * p.c.page + 15) / 16 * p.c.hkv *
                               ((static_cast<long long>(tokens) * (heads_q / p.c.hkv) + 7) / 8) * p.c.batch;
  if (heads_q > 65536 || most_tiles > 0x7fffffffLL) return fail(TOKMIX_ERR_UNSUPPORTED, "%s: problem too large", who);
  if (const int rc = check_device()) return rc;
  const long long need = tokmix_kv8_attention_workspace_bytes(tokens, heads_q, cache->heads_kv, cache->head_dim);
  if (workspace_bytes < need)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: workspace of %lld bytes, %lld needed", who, workspace_bytes, need);
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
  if (cache->head_dim == 64) return dispatch_attn<64>(who, p, e4m3, sms, workspace, s);
  if (cache->head_dim == 128) return dispatch_attn<128>(who, p, e4m3, sms, workspace, s);
  return dispatch_attn<256>(who, p, e4m3, sms, workspace, s);
}
