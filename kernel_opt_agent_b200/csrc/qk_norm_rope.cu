// qk_norm_rope.cu -- RMS norm of every query and key head with the position rotation in the same
// pass, and its gradient (sm_100a).
//
// Forward, for a head row x of D columns with weight w (the queries' or the keys'):
//   n = x / sqrt(mean x^2 + eps) * w
//   y_j = n_j cos - n_{j+half} sin,  y_{j+half} = n_j sin + n_{j+half} cos     (2 half columns behind `nope`)
// the row of the cos and sin tables named by the token's position, with several position axes that of the
// pair's axis.  All arithmetic in fp32, one rounding at the end.
// Backward, with r = 1 / sqrt(mean x^2 + eps) and g = dy turned back (the rotation's transpose):
//   dw = sum over rows of g x r,   dx = r (g w - x r^2 mean(g w x))
//
// Both are streams: a few flops per byte, bound by HBM (forward 4 bytes an element, backward 6) or, for
// few rows, by latency; next to HBM stand the issue slots, so values are computed in pairs.  A row lies in
// D / 8 lanes, 8 columns (16 bytes) each, so a warp holds 32 / (D / 8) heads of a token at a time (an iteration); sums are butterflies over a row's lanes.  Every warp takes an equal share of all
// iterations, token by token: the cos and sin of its columns are read once per token and serve its heads.
// The rows come through a ring of kDepth iterations per warp in shared memory (cp.async, each lane its own 16
// bytes), which runs ahead across tokens: what is in flight costs no registers (with loads into registers, 16 warps of 100
// registers, B4 S8192 Hq32 Hkv8 D128 ran at 4.4 TB/s), and the other half of a pair is read from the ring.
// The weights' gradients: a lane adds up its columns in registers over all its rows, a CTA adds its
// warps' sums in order and writes them to its row of a workspace, and a second launch adds those rows in
// order: the same bits every time, no atomics.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "host_common.h"
#include "sm100.cuh"

namespace tokmix {
namespace qkr {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxPairs = 128;

struct Rows {
  const void* x;             // q or k
  const void* dy;            // gradient of the output (backward)
  void* out;                 // the output, or the gradient of x: contiguous [tokens, heads, D]
  const void* w;
  long long sb, ss, sh;      // element strides of x (batch, token, head)
  long long gb, gs, gh;      // and of dy
  int heads;
};

struct Params {
  Rows q, k;
  const float *cos, *sin;    // [table_rows, half]
  const int32_t* positions;  // [axes, tokens], or null: the token's index in its sequence
  float* partial;            // backward: [CTAs, 2, D]
  long long tokens, iters;   // tokens fit 32 bits
  int seq;
  int q_iters, k_iters;      // iterations of a token: 256 / D heads each
  int half, nope, axes, table_rows;
  int w_fp32;
  float eps;
  uint32_t* status;
  uint16_t axis[kMaxPairs / 8];  // the axes of each 8 pairs, two bits a pair (axes > 1)
};

template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<__half2*>(&v));
}
template <typename T>
__device__ __forceinline__ uint32_t pack(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float a, float b) {
  return pack_bf16x2(a, b);
}
template <>
__device__ __forceinline__ uint32_t pack<__half>(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}

template <typename T>
__device__ __forceinline__ void widen(const uint4& v, F2 (&x)[4]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = unpack<T>(u[e]);
    x[e] = pair2(f.x, f.y);
  }
}

template <typename T>
__device__ __forceinline__ uint4 narrow(const F2 (&x)[4]) {
  uint32_t u[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = split2(x[e]);
    u[e] = pack<T>(f.x, f.y);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// A lane's place in its row: columns 8 part .. 8 part + 7, rotated or not, in the first or the second half of
// its pairs, and the lane that holds the other half.
struct Place {
  int part, row;       // piece of the row, row of the warp
  bool rot, first;
  int pair0;           // first pair of the 8
  int partner;         // the lane itself where nothing is rotated
  uint32_t axes;       // of the 8 pairs, two bits each
};

template <int D>
__device__ __forceinline__ Place place(const Params& p) {
  const int half = p.half, nope = p.nope;
  constexpr int kLanes = D / 8;
  const int lane = static_cast<int>(lane_id());
  Place a;
  a.part = lane % kLanes;
  a.row = lane / kLanes;
  const int v = a.part - nope / 8, hv = half / 8;
  a.rot = v >= 0 && v < 2 * hv;
  a.first = v < hv;
  a.pair0 = a.rot ? 8 * (a.first ? v : v - hv) : 0;
  a.partner = a.rot ? (a.first ? lane + hv : lane - hv) : lane;
  a.axes = p.axis[a.pair0 / 8];
  return a;
}

// The table rows of a token's axes (its index s in its sequence without positions).  Asked for a token ahead: the
// tables wait for them.
__device__ __forceinline__ int4 load_rows(const Params& p, unsigned token, unsigned s) {
  int4 r = make_int4(static_cast<int>(s), 0, 0, 0);
  if (p.positions != nullptr && token < p.tokens) {
    const int32_t* at = p.positions + token;
    r.x = __ldg(at);
    if (p.axes > 1) r.y = __ldg(at + p.tokens);
    if (p.axes > 2) r.z = __ldg(at + 2 * p.tokens);
    if (p.axes > 3) r.w = __ldg(at + 3 * p.tokens);
  }
  return r;
}

// cos and sin of the lane's 8 pairs; 1 and 0 where nothing is rotated, NaN (and a status bit) where a
// position lies outside the tables.  sin is negated for the first half, so that y = n cos + n_partner sin
// in both.
__device__ __forceinline__ void load_turn(const Params& p, const Place& a, const int4& row, float (&c)[8], float (&s)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    c[e] = 1.0f;
    s[e] = 0.0f;
  }
  if (!a.rot) return;
  const unsigned rows = static_cast<unsigned>(p.table_rows);
  if (static_cast<unsigned>(row.x) >= rows || static_cast<unsigned>(row.y) >= rows || static_cast<unsigned>(row.z) >= rows ||
      static_cast<unsigned>(row.w) >= rows) {
    record_status(p.status, kDevBadArgs);
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = s[e] = __int_as_float(0x7fffffff);
  } else if (p.axes <= 1) {
    const long long at = static_cast<long long>(row.x) * p.half + a.pair0;
    const float4* cp = reinterpret_cast<const float4*>(p.cos + at);
    const float4* sp = reinterpret_cast<const float4*>(p.sin + at);
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const float4 cv = __ldg(cp + v), sv = __ldg(sp + v);
      c[4 * v] = cv.x; c[4 * v + 1] = cv.y; c[4 * v + 2] = cv.z; c[4 * v + 3] = cv.w;
      s[4 * v] = sv.x; s[4 * v + 1] = sv.y; s[4 * v + 2] = sv.z; s[4 * v + 3] = sv.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t x = a.axes >> (2 * e) & 3u;
      const long long at = static_cast<long long>(x == 0 ? row.x : x == 1 ? row.y : x == 2 ? row.z : row.w) * p.half + a.pair0 + e;
      c[e] = __ldg(p.cos + at);
      s[e] = __ldg(p.sin + at);
    }
  }
  if (a.first) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = -s[e];
  }
}

template <typename T>
__device__ __forceinline__ void stage_weights(const Params& p, int d, float* w) {
  for (int i = threadIdx.x; i < 2 * d; i += kThreads) {
    const void* src = i < d ? p.q.w : p.k.w;
    const int c = i < d ? i : i - d;
    w[i] = p.w_fp32 ? static_cast<const float*>(src)[c] : static_cast<float>(static_cast<const T*>(src)[c]);
  }
  __syncthreads();
}

// A place in the sequence of all iterations, token by token, the queries' of a token before its keys'.
// Every warp takes an equal share of the sequence, which may begin and end inside a token.
struct Spot {
  unsigned token, b, s;
  int it;            // iteration of the token
  long long left;    // iterations to the end of the warp's share

  __device__ __forceinline__ void begin(const Params& p) {
    const long long warps = static_cast<long long>(gridDim.x) * kWarps, w = static_cast<long long>(blockIdx.x) * kWarps + warp_id();
    const int per = p.q_iters + p.k_iters;
    const long long lo = p.iters / warps * w + min(w, p.iters % warps);
    left = p.iters / warps + (w < p.iters % warps ? 1 : 0);
    token = static_cast<unsigned>(lo / per);
    it = static_cast<int>(lo - static_cast<long long>(token) * per);
    b = token / static_cast<unsigned>(p.seq);
    s = token - b * static_cast<unsigned>(p.seq);
  }
  __device__ __forceinline__ void next_token(const Params& p) {
    it = 0;
    ++token;
    if (++s == static_cast<unsigned>(p.seq)) {
      s = 0;
      ++b;
    }
  }
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The warp ahead of its work: copies iteration after iteration into the ring.
template <int D, typename T, bool kBackward>
struct Ahead {
  static constexpr int kRows = 256 / D;
  Spot at;
  int until;                  // iterations of this kind left in the token
  int h, heads;               // this lane's head in the iteration, heads of the kind
  const T *x, *g;             // its 16 bytes
  long long x_step, g_step;   // to the next iteration's

  __device__ __forceinline__ void point(const Params& p, const Place& a) {
    const bool is_q = at.it < p.q_iters;
    const Rows& r = is_q ? p.q : p.k;
    const int first = is_q ? at.it : at.it - p.q_iters;
    until = (is_q ? p.q_iters : p.k_iters) - first;
    h = first * kRows + a.row;
    heads = r.heads;
    x = static_cast<const T*>(r.x) + at.b * r.sb + at.s * r.ss + h * r.sh + a.part * 8;
    x_step = r.sh * kRows;
    if (kBackward) {
      g = static_cast<const T*>(r.dy) + at.b * r.gb + at.s * r.gs + h * r.gh + a.part * 8;
      g_step = r.gh * kRows;
    }
  }
  __device__ __forceinline__ void begin(const Params& p, const Place& a) {
    at.begin(p);
    if (at.left > 0) point(p, a);
  }
  __device__ __forceinline__ void fetch(const Params& p, const Place& a, uint32_t slot) {
    if (at.left > 0) {
      copy16(slot, x, h < heads);
      if (kBackward) copy16(slot + 512, g, h < heads);
      x += x_step;
      if (kBackward) g += g_step;
      h += kRows;
      ++at.it;
      --at.left;
      if (--until == 0 && at.left > 0) {
        if (at.it == p.q_iters + p.k_iters) at.next_token(p);
        point(p, a);
      }
    }
    copy_commit();
  }
};

__device__ __forceinline__ uint4 ring_read(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// Iterations in flight per warp: enough to cover the way to memory; deeper rings only lengthen the start and the end.  Forward
// B4 S8192 Hq32 Hkv8 D128 118 us at 5, 115.8 at 6, 114.3 at 8, 115.5 at 10; gradient B2 S4096 Hq16 Hkv2 D256, three axes, 46.8 at 3,
// 46.3 at 4, 46.7 at 5, 47.7 at 8, 48.7 at 10, B4 S8192 Hq32 Hkv8 D128 on two inputs in turn 174 at 4, 169 at 5, 173 at 8 and 10.
constexpr int kFwdDepth = 8, kBwdDepth = 5;
constexpr int kFwdPerSm = 2, kBwdPerSm = 2;  // CTAs

template <int D, typename T>
__global__ void __launch_bounds__(kThreads, kFwdPerSm) qk_norm_rope_kernel(const __grid_constant__ Params p) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;
  __shared__ __align__(16) float w[2 * D];
  __shared__ __align__(16) uint8_t ring_mem[kWarps][kFwdDepth * 512];
  wait_previous_kernels();
  stage_weights<T>(p, D, w);
  const Place a = place<D>(p);
  const int partner_part = a.partner % kLanes;
  const uint32_t ring = smem_u32(ring_mem[warp_id()]);
  const uint32_t own = lane_id() * 16, other = a.partner * 16;
  Ahead<D, T, false> ahead;
  ahead.begin(p, a);
  Spot c = ahead.at;
  int4 rows = load_rows(p, c.token, c.s);
#pragma unroll 1
  for (int i = 0; i < kFwdDepth; ++i) ahead.fetch(p, a, ring + i * 512 + own);
  uint32_t slot = ring;
  for (; c.left > 0; c.next_token(p)) {
    const int end = static_cast<int>(min(static_cast<long long>(p.q_iters + p.k_iters), c.it + c.left));
    c.left -= end - c.it;
    float cs[8], sn[8];
    load_turn(p, a, rows, cs, sn);
    rows = load_rows(p, c.token + 1, c.s + 1 == static_cast<unsigned>(p.seq) ? 0u : c.s + 1);
#pragma unroll 1
    for (int kind = 0; kind < 2; ++kind) {
      const Rows& r = kind ? p.k : p.q;
      const int lo = kind ? max(c.it - p.q_iters, 0) : c.it;
      const int hi = kind ? end - p.q_iters : min(end, p.q_iters);
      if (lo >= hi) continue;
      int h = lo * kRows + a.row;
      T* dst = static_cast<T*>(r.out) + (static_cast<long long>(c.token) * r.heads + h) * D + a.part * 8;
      // own weights times cos, the partner's times sin: y = r (x (w cos) + x_partner (w_partner sin)); where nothing is
      // rotated the partner is the lane itself and sin 0
      const float *wo = w + kind * D + a.part * 8, *wp = w + kind * D + partner_part * 8;
      F2 wc[4], ws[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        wc[e] = pair2(wo[2 * e] * cs[2 * e], wo[2 * e + 1] * cs[2 * e + 1]);
        ws[e] = pair2(wp[2 * e] * sn[2 * e], wp[2 * e + 1] * sn[2 * e + 1]);
      }
#pragma unroll 1
      for (int left = hi - lo; left > 0; --left, h += kRows, dst += kRows * D) {
        copy_wait<kFwdDepth - 1>();
        __syncwarp();
        F2 x[4], o[4];
        widen<T>(ring_read(slot + own), x);
        widen<T>(ring_read(slot + other), o);
        __syncwarp();
        ahead.fetch(p, a, slot + own);
        slot = slot == ring + (kFwdDepth - 1) * 512 ? ring : slot + 512;
        F2 sq = mul2(x[0], x[0]);
#pragma unroll
        for (int e = 1; e < 4; ++e) sq = fma2(x[e], x[e], sq);
        float sum = split2(sq).x + split2(sq).y;
#pragma unroll
        for (int m = kLanes / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
        const float inv = rsqrtf(sum * (1.0f / D) + p.eps);
        const F2 inv2 = pair2(inv, inv);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = mul2(inv2, fma2(o[e], ws[e], mul2(x[e], wc[e])));
        if (h < r.heads) *reinterpret_cast<uint4*>(dst) = narrow<T>(x);
      }
    }
  }
}

template <int D, typename T>
__global__ void __launch_bounds__(kThreads, kBwdPerSm) qk_norm_rope_bwd_kernel(const __grid_constant__ Params p) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;
  extern __shared__ __align__(16) uint8_t dyn[];  // the rings: [kWarps][kBwdDepth][x, dy][512]
  __shared__ __align__(16) float w[2 * D];
  wait_previous_kernels();
  stage_weights<T>(p, D, w);
  const Place a = place<D>(p);
  F2 acc[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = 0ull;
  const uint32_t ring = smem_u32(dyn) + warp_id() * (kBwdDepth * 1024);
  const uint32_t own = lane_id() * 16, other = a.partner * 16;
  Ahead<D, T, true> ahead;
  ahead.begin(p, a);
  Spot c = ahead.at;
  int4 rows = load_rows(p, c.token, c.s);
#pragma unroll 1
  for (int i = 0; i < kBwdDepth; ++i) ahead.fetch(p, a, ring + i * 1024 + own);
  uint32_t slot = ring;
  for (; c.left > 0; c.next_token(p)) {
    const int end = static_cast<int>(min(static_cast<long long>(p.q_iters + p.k_iters), c.it + c.left));
    c.left -= end - c.it;
    F2 c2[4], s2[4];
    {
      float cs[8], sn[8];
      load_turn(p, a, rows, cs, sn);
      rows = load_rows(p, c.token + 1, c.s + 1 == static_cast<unsigned>(p.seq) ? 0u : c.s + 1);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c2[e] = pair2(cs[2 * e], cs[2 * e + 1]);
        s2[e] = pair2(-sn[2 * e], -sn[2 * e + 1]);
      }
    }
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const Rows& r = kind ? p.k : p.q;
      const int lo = kind ? max(c.it - p.q_iters, 0) : c.it;
      const int hi = kind ? end - p.q_iters : min(end, p.q_iters);
      if (lo >= hi) continue;
      int h = lo * kRows + a.row;
      T* dst = static_cast<T*>(r.out) + (static_cast<long long>(c.token) * r.heads + h) * D + a.part * 8;
      const F2* wo = reinterpret_cast<const F2*>(w + kind * D + a.part * 8);
      F2 wl[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) wl[e] = wo[e];
#pragma unroll 1
      for (int left = hi - lo; left > 0; --left, h += kRows, dst += kRows * D) {
        copy_wait<kBwdDepth - 1>();
        __syncwarp();
        F2 x[4], g[4], o[4];
        widen<T>(ring_read(slot + own), x);
        widen<T>(ring_read(slot + 512 + own), g);
        widen<T>(ring_read(slot + 512 + other), o);
        __syncwarp();
        ahead.fetch(p, a, slot + own);
        slot = slot == ring + (kBwdDepth - 1) * 1024 ? ring : slot + 1024;
        F2 sq = 0ull, gx = 0ull;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          g[e] = fma2(o[e], s2[e], mul2(g[e], c2[e]));  // turned back
          o[e] = mul2(g[e], wl[e]);
          sq = fma2(x[e], x[e], sq);
          gx = fma2(o[e], x[e], gx);
        }
        float sum = split2(sq).x + split2(sq).y, dot = split2(gx).x + split2(gx).y;
#pragma unroll
        for (int m = kLanes / 2; m > 0; m >>= 1) {
          sum += __shfl_xor_sync(0xffffffffu, sum, m);
          dot += __shfl_xor_sync(0xffffffffu, dot, m);
        }
        // Where the iteration has no head, its zeros would, without eps, add 0 * inf to the weights' sums.  Chosen here, before the
        // sum is there, it takes no time: B2 S4096 Hq16 Hkv2 D256, three axes, 45.8 us (45.7 without it, 46.4 chosen behind the root).
        const float inv = rsqrtf(fmaf(sum, 1.0f / D, h < r.heads ? p.eps : 1.0f));
        // x r before r again: without eps, r^2 alone passes fp32's range where x r^2 does not
        const float back = -inv * (dot * (1.0f / D));
        const F2 inv2 = pair2(inv, inv), back2 = pair2(back, back);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = mul2(x[e], inv2);
          acc[kind][e] = fma2(g[e], x[e], acc[kind][e]);
          x[e] = mul2(inv2, fma2(back2, x[e], o[e]));
        }
        if (h < r.heads) *reinterpret_cast<uint4*>(dst) = narrow<T>(x);
      }
    }
  }
  // the warp's rows, then the CTA's warps in order (over the rings)
  copy_wait<0>();
  __syncthreads();
  float* sums = reinterpret_cast<float*>(dyn);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float t = e % 2 ? split2(acc[i][e / 2]).y : split2(acc[i][e / 2]).x;
#pragma unroll
      for (int m = kLanes; m < 32; m <<= 1) t += __shfl_xor_sync(0xffffffffu, t, m);
      if (a.row == 0) sums[warp_id() * 2 * D + i * D + a.part * 8 + e] = t;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
    float t = 0.0f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) t += sums[v * 2 * D + i];
    p.partial[static_cast<long long>(blockIdx.x) * 2 * D + i] = t;
  }
}
constexpr int kBwdSmem = kWarps * kBwdDepth * 1024;
static_assert(kBwdSmem >= kWarps * 2 * 256 * 4, "the warps' sums fit where the rings were");

// dw[i] = the sum of the CTAs' rows in order: 32 columns a block, each by 32 threads that take every
// 32nd row, joined in order.  Rounded to the weights' type.
template <typename T>
__global__ void __launch_bounds__(1024) weight_grad_kernel(const float* __restrict__ partial, int rows, int d, T* __restrict__ dwq,
                                                           T* __restrict__ dwk) {
  __shared__ float sums[32][33];
  wait_previous_kernels();
  const int col = blockIdx.x * 32 + threadIdx.x;  // 2 d columns: the queries' weight, the keys'
  float t = 0.0f;
  for (int r = threadIdx.y; r < rows; r += 32) t += partial[static_cast<long long>(r) * 2 * d + col];
  sums[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.y == 0) {
    t = 0.0f;
#pragma unroll
    for (int v = 0; v < 32; ++v) t += sums[v][threadIdx.x];
    if (col < d)
      dwq[col] = static_cast<T>(t);
    else
      dwk[col - d] = static_cast<T>(t);
  }
}

// CTAs of a call: `per_sm` to an SM (its registers), fewer where warps would have no iteration.
int ctas(long long iters, int per_sm) {
  return static_cast<int>(std::min<long long>((iters + kWarps - 1) / kWarps, static_cast<long long>(per_sm) * std::max(1, device_sm_count())));
}

int iterations(int heads, int d) { return (heads + 256 / d - 1) / (256 / d); }

template <int D, typename T>
cudaError_t run_fwd(const Params& p, cudaStream_t stream) {
  return launch_overlapped(&qk_norm_rope_kernel<D, T>, dim3(static_cast<unsigned>(ctas(p.iters, kFwdPerSm))), dim3(kThreads), 0, stream,
                           p);
}

template <int D, typename T>
cudaError_t run_bwd(const Params& p, void* dwq, void* dwk, cudaStream_t stream) {
  const int rows = ctas(p.iters, kBwdPerSm);
  if (!ensure_smem_attr(reinterpret_cast<const void*>(&qk_norm_rope_bwd_kernel<D, T>), kBwdSmem)) return cudaGetLastError();
  const cudaError_t e = launch_overlapped(&qk_norm_rope_bwd_kernel<D, T>, dim3(static_cast<unsigned>(rows)), dim3(kThreads),
                                          static_cast<size_t>(kBwdSmem), stream, p);
  if (e != cudaSuccess) return e;
  const dim3 blocks(2 * D / 32), threads(32, 32);
  if (p.w_fp32)
    return launch_overlapped(&weight_grad_kernel<float>, blocks, threads, 0, stream, p.partial, rows, D, static_cast<float*>(dwq),
                             static_cast<float*>(dwk));
  return launch_overlapped(&weight_grad_kernel<T>, blocks, threads, 0, stream, p.partial, rows, D, static_cast<T*>(dwq),
                           static_cast<T*>(dwk));
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Checks shared by both directions; fills p.
int prepare(const char* who, const tokmix_qk_norm_rope* a, bool backward, Params& p) {
  if (a == nullptr) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: null description", who);
  if (a->batch < 0 || a->seqlen < 0 || a->heads_q <= 0 || a->heads_k <= 0)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: negative or zero size", who);
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256)
    return fail(TOKMIX_ERR_UNSUPPORTED, "%s: head_dim %d not supported (64, 128 or 256)", who, a->head_dim);
  if ((a->dtype != TOKMIX_DTYPE_BF16 && a->dtype != TOKMIX_DTYPE_FP16) ||
      (a->weight_dtype != a->dtype && a->weight_dtype != TOKMIX_DTYPE_FP32))
    return fail(TOKMIX_ERR_UNSUPPORTED, "%s: bf16 or fp16 tensors with weights of that type or fp32", who);
  if (a->half <= 0 || a->half % 8 != 0 || a->nope < 0 || a->nope % 8 != 0 || a->nope + 2 * a->half > a->head_dim)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: half and nope must be multiples of 8 with nope + 2 half <= head_dim", who);
  p.tokens = static_cast<long long>(a->batch) * a->seqlen;  // without any, positions may be an empty tensor's address, null
  if (a->axes < 1 || a->axes > 4 || (a->axes > 1 && ((a->positions == nullptr && p.tokens > 0) || a->pair_axis == nullptr)))
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: 1 to 4 position axes; several need positions and an axis per pair", who);
  if (!(a->eps >= 0.0f) || !std::isfinite(a->eps)) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: eps must be finite and not negative", who);
  if (a->table_rows <= 0 || (a->positions == nullptr && p.tokens > 0 && a->table_rows < a->seqlen))
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: the tables must have a row for every position", who);
  for (const long long s : {a->q_batch_stride, a->q_token_stride, a->q_head_stride, a->k_batch_stride, a->k_token_stride,
                            a->k_head_stride})
    if (s % 8 != 0) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: strides must be multiples of 8 elements", who);
  if (backward)
    for (const long long s : {a->dq_batch_stride, a->dq_token_stride, a->dq_head_stride, a->dk_batch_stride, a->dk_token_stride,
                              a->dk_head_stride})
      if (s % 8 != 0) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: strides must be multiples of 8 elements", who);
  if (p.tokens > 0x7FFFFFFFll) return fail(TOKMIX_ERR_UNSUPPORTED, "%s: too many tokens (%lld)", who, p.tokens);
  if (a->heads_q > 65536 || a->heads_k > 65536) return fail(TOKMIX_ERR_UNSUPPORTED, "%s: more than 65536 heads", who);
  if (p.tokens == 0 && !backward) return TOKMIX_OK;
  if (a->q_weight == nullptr || a->k_weight == nullptr)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: null weight", who);
  if (p.tokens > 0) {
    for (const void* t : {a->q, a->k, static_cast<const void*>(a->q_out), static_cast<const void*>(a->k_out),
                          static_cast<const void*>(a->cos), static_cast<const void*>(a->sin)})
      if (t == nullptr || !aligned16(t))
        return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: tensors must be non-null and 16-byte aligned", who);
    if (backward && (a->dq == nullptr || a->dk == nullptr || !aligned16(a->dq) || !aligned16(a->dk)))
      return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: gradients must be non-null and 16-byte aligned", who);
  }
  p.q = Rows{a->q, a->dq, a->q_out, a->q_weight, a->q_batch_stride, a->q_token_stride, a->q_head_stride,
             a->dq_batch_stride, a->dq_token_stride, a->dq_head_stride, a->heads_q};
  p.k = Rows{a->k, a->dk, a->k_out, a->k_weight, a->k_batch_stride, a->k_token_stride, a->k_head_stride,
             a->dk_batch_stride, a->dk_token_stride, a->dk_head_stride, a->heads_k};
  p.cos = a->cos;
  p.sin = a->sin;
  p.positions = a->positions;
  p.seq = std::max(1, a->seqlen);
  p.q_iters = iterations(a->heads_q, a->head_dim);
  p.k_iters = iterations(a->heads_k, a->head_dim);
  p.iters = p.tokens * (p.q_iters + p.k_iters);
  p.half = a->half;
  p.nope = a->nope;
  p.axes = a->axes;
  p.table_rows = a->table_rows;
  p.w_fp32 = a->weight_dtype == TOKMIX_DTYPE_FP32 ? 1 : 0;
  p.eps = a->eps;
  for (int i = 0; i < a->half; ++i) {
    const int x = a->axes > 1 ? a->pair_axis[i] : 0;
    if (x >= a->axes) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: pair %d names axis %d of %d", who, i, x, a->axes);
    p.axis[i / 8] = static_cast<uint16_t>(p.axis[i / 8] | x << (2 * (i % 8)));
  }
  return TOKMIX_OK;
}

}  // namespace qkr
}  // namespace tokmix

extern "C" int tokmix_qk_norm_rope_fwd(const tokmix_qk_norm_rope* a, uint32_t* status, void* stream) {
  using namespace tokmix;
  qkr::Params p{};
  if (const int rc = qkr::prepare("tokmix_qk_norm_rope_fwd", a, false, p)) return rc;
  if (p.tokens == 0) return TOKMIX_OK;
  if (const int rc = check_device()) return rc;
  p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = a->dtype == TOKMIX_DTYPE_BF16;
  cudaError_t e;
  if (a->head_dim == 64)
    e = bf16 ? qkr::run_fwd<64, __nv_bfloat16>(p, s) : qkr::run_fwd<64, __half>(p, s);
  else if (a->head_dim == 128)
    e = bf16 ? qkr::run_fwd<128, __nv_bfloat16>(p, s) : qkr::run_fwd<128, __half>(p, s);
  else
    e = bf16 ? qkr::run_fwd<256, __nv_bfloat16>(p, s) : qkr::run_fwd<256, __half>(p, s);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(TOKMIX_ERR_LAUNCH, "tokmix_qk_norm_rope_fwd: %s", cudaGetErrorString(e));
  }
  return check_launch("tokmix_qk_norm_rope_fwd");
}

extern "C" long long tokmix_qk_norm_rope_bwd_workspace_bytes(long long tokens, int heads_q, int heads_k, int head_dim) {
  using namespace tokmix;
  if (tokens < 0 || heads_q <= 0 || heads_k <= 0 || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return -1;
  const long long iters = tokens * (qkr::iterations(heads_q, head_dim) + qkr::iterations(heads_k, head_dim));
  return static_cast<long long>(qkr::ctas(iters, qkr::kBwdPerSm)) * 2 * head_dim * 4;
}

extern "C" int tokmix_qk_norm_rope_bwd(const tokmix_qk_norm_rope* a, void* dq_weight, void* dk_weight, void* workspace,
                                       long long workspace_bytes, uint32_t* status, void* stream) {
  using namespace tokmix;
  qkr::Params p{};
  if (const int rc = qkr::prepare("tokmix_qk_norm_rope_bwd", a, true, p)) return rc;
  if (dq_weight == nullptr || dk_weight == nullptr)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_qk_norm_rope_bwd: null weight gradient");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (const int rc = check_device()) return rc;
  if (p.tokens == 0) {
    const size_t bytes = static_cast<size_t>(a->head_dim) * (a->weight_dtype == TOKMIX_DTYPE_FP32 ? 4 : 2);
    if (cudaMemsetAsync(dq_weight, 0, bytes, s) != cudaSuccess || cudaMemsetAsync(dk_weight, 0, bytes, s) != cudaSuccess)
      return check_launch("tokmix_qk_norm_rope_bwd");
    return TOKMIX_OK;
  }
  const long long need = tokmix_qk_norm_rope_bwd_workspace_bytes(p.tokens, a->heads_q, a->heads_k, a->head_dim);
  if (workspace == nullptr || workspace_bytes < need || !qkr::aligned16(workspace))
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_qk_norm_rope_bwd: needs a 16-byte aligned workspace of %lld bytes", need);
  p.partial = static_cast<float*>(workspace);
  p.status = status;
  const bool bf16 = a->dtype == TOKMIX_DTYPE_BF16;
  cudaError_t e;
  if (a->head_dim == 64)
    e = bf16 ? qkr::run_bwd<64, __nv_bfloat16>(p, dq_weight, dk_weight, s) : qkr::run_bwd<64, __half>(p, dq_weight, dk_weight, s);
  else if (a->head_dim == 128)
    e = bf16 ? qkr::run_bwd<128, __nv_bfloat16>(p, dq_weight, dk_weight, s) : qkr::run_bwd<128, __half>(p, dq_weight, dk_weight, s);
  else
    e = bf16 ? qkr::run_bwd<256, __nv_bfloat16>(p, dq_weight, dk_weight, s) : qkr::run_bwd<256, __half>(p, dq_weight, dk_weight, s);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(TOKMIX_ERR_LAUNCH, "tokmix_qk_norm_rope_bwd: %s", cudaGetErrorString(e));
  }
  return check_launch("tokmix_qk_norm_rope_bwd");
}
