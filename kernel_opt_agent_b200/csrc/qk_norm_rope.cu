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
// few rows, by latency.  A row lies in D / 8 lanes, 8 columns (16 bytes) each, so a warp holds 32 / (D / 8) heads
// of a token; sums are butterflies over a row's lanes, and the other half of a pair comes from the lane half / 8
// away.  A warp takes a token (or, when tokens are few, a part of its heads): the cos and sin of its
// columns are read once and serve all heads, and the loads of `U` rows are issued before the first
// is used.
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
  long long tokens, units;
  int seq, parts;            // a unit is one of `parts` parts of a token's heads
  int half, nope, axes, table_rows;
  int w_fp32;
  float eps;
  uint32_t* status;
  uint8_t axis[kMaxPairs];   // the axis of each pair (axes > 1)
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
__device__ __forceinline__ void widen(const uint4& v, float (&x)[8]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = unpack<T>(u[e]);
    x[2 * e] = f.x;
    x[2 * e + 1] = f.y;
  }
}

template <typename T>
__device__ __forceinline__ uint4 narrow(const float (&x)[8]) {
  return make_uint4(pack<T>(x[0], x[1]), pack<T>(x[2], x[3]), pack<T>(x[4], x[5]), pack<T>(x[6], x[7]));
}

__device__ __forceinline__ uint4 shfl4(const uint4& v, int src) {
  return make_uint4(__shfl_sync(0xffffffffu, v.x, src), __shfl_sync(0xffffffffu, v.y, src),
                    __shfl_sync(0xffffffffu, v.z, src), __shfl_sync(0xffffffffu, v.w, src));
}

// A lane's place in its row: columns 8 part .. 8 part + 7, rotated or not, in the first or the second half of
// its pairs, and the lane that holds the other half.
struct Place {
  int part, row;       // piece of the row, row of the warp
  bool rot, first;
  int pair0;           // first pair of the 8
  int partner;
};

template <int D>
__device__ __forceinline__ Place place(int half, int nope) {
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
  return a;
}

// cos and sin of the lane's 8 pairs at token t; 1 and 0 where nothing is rotated, NaN (and a status
// bit) where a position lies outside the tables.  sin is negated for the first half, so that
// y = n cos + n_partner sin in both.
__device__ __forceinline__ void load_turn(const Params& p, const Place& a, long long t, float (&c)[8], float (&s)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    c[e] = 1.0f;
    s[e] = 0.0f;
  }
  if (!a.rot) return;
  bool bad = false;
  if (p.axes <= 1) {
    const long long row = p.positions != nullptr ? p.positions[t] : t % p.seq;
    bad = row < 0 || row >= p.table_rows;
    if (!bad) {
      const float4* cp = reinterpret_cast<const float4*>(p.cos + row * p.half + a.pair0);
      const float4* sp = reinterpret_cast<const float4*>(p.sin + row * p.half + a.pair0);
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const float4 cv = __ldg(cp + v), sv = __ldg(sp + v);
        c[4 * v] = cv.x; c[4 * v + 1] = cv.y; c[4 * v + 2] = cv.z; c[4 * v + 3] = cv.w;
        s[4 * v] = sv.x; s[4 * v + 1] = sv.y; s[4 * v + 2] = sv.z; s[4 * v + 3] = sv.w;
      }
    }
  } else {
    long long row[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      row[x] = x < p.axes ? p.positions[x * p.tokens + t] : 0;
      bad = bad || row[x] < 0 || row[x] >= p.table_rows;
    }
    if (!bad) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int x = p.axis[a.pair0 + e];
        const long long at = (x == 0 ? row[0] : x == 1 ? row[1] : x == 2 ? row[2] : row[3]) * p.half + a.pair0 + e;
        c[e] = __ldg(p.cos + at);
        s[e] = __ldg(p.sin + at);
      }
    }
  }
  if (bad) {
    record_status(p.status, kDevBadArgs);
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = s[e] = __int_as_float(0x7fffffff);
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

// The rows [lo, hi) of iterations of a unit, one iteration being 32 / (D / 8) heads; the queries' come first.
struct Range {
  long long token;
  int q_lo, q_hi, k_lo, k_hi;
};

template <int D>
__device__ __forceinline__ Range unit_range(const Params& p, long long u) {
  constexpr int kRows = 256 / D;
  const int nq = (p.q.heads + kRows - 1) / kRows, nk = (p.k.heads + kRows - 1) / kRows;
  Range r;
  r.token = u / p.parts;
  const int part = static_cast<int>(u - r.token * p.parts);
  const int lo = static_cast<int>(static_cast<long long>(nq + nk) * part / p.parts);
  const int hi = static_cast<int>(static_cast<long long>(nq + nk) * (part + 1) / p.parts);
  r.q_lo = min(lo, nq);
  r.q_hi = min(hi, nq);
  r.k_lo = max(lo, nq) - nq;
  r.k_hi = max(hi, nq) - nq;
  return r;
}

template <int D, typename T, int U>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const __grid_constant__ Params p) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;
  __shared__ __align__(16) float w[2 * D];
  wait_previous_kernels();
  stage_weights<T>(p, D, w);
  const Place a = place<D>(p.half, p.nope);
  const int partner_part = a.partner % kLanes;
  const long long stride = static_cast<long long>(gridDim.x) * kWarps;
  for (long long u = static_cast<long long>(blockIdx.x) * kWarps + warp_id(); u < p.units; u += stride) {
    const Range rg = unit_range<D>(p, u);
    const long long b = rg.token / p.seq, s = rg.token - b * p.seq;
    float c[8], sn[8];
    load_turn(p, a, rg.token, c, sn);
    auto rows = [&](const Rows& r, const float* wr, int lo, int hi) {
      if (lo >= hi) return;
      const T* src = static_cast<const T*>(r.x) + b * r.sb + s * r.ss + a.part * 8;
      T* dst = static_cast<T*>(r.out) + rg.token * r.heads * D + a.part * 8;
      // own weights times cos, the partner's times sin: y = r (x (w cos) + x_partner (w_partner sin))
      float wc[8], ws[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        wc[e] = wr[a.part * 8 + e] * c[e];
        ws[e] = wr[partner_part * 8 + e] * sn[e];
      }
      for (int it = lo; it < hi; it += U) {
        uint4 v[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const int h = (it + k) * kRows + a.row;
          v[k] = it + k < hi && h < r.heads ? __ldcs(reinterpret_cast<const uint4*>(src + h * r.sh)) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
          if (it + k >= hi) break;  // warp-uniform
          const int h = (it + k) * kRows + a.row;
          float x[8], o[8];
          widen<T>(v[k], x);
          widen<T>(shfl4(v[k], a.partner), o);
          float sum = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
          for (int m = kLanes / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
          const float inv = rsqrtf(sum * (1.0f / D) + p.eps);
          // an unrotated lane has no second term (0 times an infinite x would be NaN)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = inv * (a.rot ? fmaf(o[e], ws[e], x[e] * wc[e]) : x[e] * wc[e]);
          if (h < r.heads) *reinterpret_cast<uint4*>(dst + h * D) = narrow<T>(x);
        }
      }
    };
    rows(p.q, w, rg.q_lo, rg.q_hi);
    rows(p.k, w + D, rg.k_lo, rg.k_hi);
  }
}

template <int D, typename T, int U>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_bwd_kernel(const __grid_constant__ Params p) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes;
  __shared__ __align__(16) float w[2 * D];
  __shared__ float sums[kWarps][2 * D];
  wait_previous_kernels();
  stage_weights<T>(p, D, w);
  const Place a = place<D>(p.half, p.nope);
  float acc[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[i][e] = 0.0f;
  const long long stride = static_cast<long long>(gridDim.x) * kWarps;
  for (long long u = static_cast<long long>(blockIdx.x) * kWarps + warp_id(); u < p.units; u += stride) {
    const Range rg = unit_range<D>(p, u);
    const long long b = rg.token / p.seq, s = rg.token - b * p.seq;
    float c[8], sn[8];
    load_turn(p, a, rg.token, c, sn);
    auto rows = [&](const Rows& r, const float* wr, float (&dw)[8], int lo, int hi) {
      if (lo >= hi) return;
      const T* src = static_cast<const T*>(r.x) + b * r.sb + s * r.ss + a.part * 8;
      const T* grad = static_cast<const T*>(r.dy) + b * r.gb + s * r.gs + a.part * 8;
      T* dst = static_cast<T*>(r.out) + rg.token * r.heads * D + a.part * 8;
      float wl[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) wl[e] = wr[a.part * 8 + e];
      for (int it = lo; it < hi; it += U) {
        uint4 v[U], dv[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const int h = (it + k) * kRows + a.row;
          const bool in = it + k < hi && h < r.heads;
          v[k] = in ? __ldcs(reinterpret_cast<const uint4*>(src + h * r.sh)) : make_uint4(0u, 0u, 0u, 0u);
          dv[k] = in ? __ldcs(reinterpret_cast<const uint4*>(grad + h * r.gh)) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
          if (it + k >= hi) break;  // warp-uniform
          const int h = (it + k) * kRows + a.row;
          float x[8], g[8], o[8];
          widen<T>(v[k], x);
          widen<T>(dv[k], g);
          widen<T>(shfl4(dv[k], a.partner), o);
          if (a.rot) {
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = fmaf(o[e], -sn[e], g[e] * c[e]);  // turned back
          }
          float sum = 0.0f, dot = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            sum = fmaf(x[e], x[e], sum);
            dot = fmaf(g[e] * wl[e], x[e], dot);
          }
#pragma unroll
          for (int m = kLanes / 2; m > 0; m >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, m);
            dot += __shfl_xor_sync(0xffffffffu, dot, m);
          }
          const float inv = rsqrtf(sum * (1.0f / D) + p.eps);
          const float back = inv * inv * (dot * (1.0f / D));
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            dw[e] = fmaf(g[e], x[e] * inv, dw[e]);
            x[e] = inv * fmaf(-back, x[e], g[e] * wl[e]);
          }
          if (h < r.heads) *reinterpret_cast<uint4*>(dst + h * D) = narrow<T>(x);
        }
      }
    };
    rows(p.q, w, acc[0], rg.q_lo, rg.q_hi);
    rows(p.k, w + D, acc[1], rg.k_lo, rg.k_hi);
  }
  // the warp's rows, then the CTA's warps in order
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
      for (int m = kLanes; m < 32; m <<= 1) acc[i][e] += __shfl_xor_sync(0xffffffffu, acc[i][e], m);
      if (a.row == 0) sums[warp_id()][i * D + a.part * 8 + e] = acc[i][e];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
    float t = 0.0f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) t += sums[v][i];
    p.partial[static_cast<long long>(blockIdx.x) * 2 * D + i] = t;
  }
}

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

// CTAs of a backward call: four to an SM (its registers), fewer where warps would have no unit.
int bwd_ctas(long long units) {
  return static_cast<int>(std::min<long long>((units + kWarps - 1) / kWarps, 4LL * std::max(1, device_sm_count())));
}

// Parts of a token's heads: as many as it takes to give every SM 32 warps, at most one per iteration.
int head_parts(long long tokens, int heads_q, int heads_k, int d) {
  const int rows = 256 / d;
  const int iters = (heads_q + rows - 1) / rows + (heads_k + rows - 1) / rows;
  const long long want = 32LL * std::max(1, device_sm_count());
  return static_cast<int>(std::max<long long>(1, std::min<long long>(iters, (want + tokens - 1) / std::max<long long>(1, tokens))));
}

template <int D, typename T>
cudaError_t run_fwd(const Params& p, cudaStream_t stream) {
  const long long ctas = std::min<long long>((p.units + kWarps - 1) / kWarps, 8LL * std::max(1, device_sm_count()));
  const dim3 grid(static_cast<unsigned>(ctas));
  if (p.parts > 1) return launch_overlapped(&qk_norm_rope_kernel<D, T, 1>, grid, dim3(kThreads), 0, stream, p);
  return launch_overlapped(&qk_norm_rope_kernel<D, T, 4>, grid, dim3(kThreads), 0, stream, p);
}

template <int D, typename T>
cudaError_t run_bwd(const Params& p, void* dwq, void* dwk, cudaStream_t stream) {
  const int ctas = bwd_ctas(p.units);
  const dim3 grid(static_cast<unsigned>(ctas));
  cudaError_t e = p.parts > 1 ? launch_overlapped(&qk_norm_rope_bwd_kernel<D, T, 1>, grid, dim3(kThreads), 0, stream, p)
                              : launch_overlapped(&qk_norm_rope_bwd_kernel<D, T, 2>, grid, dim3(kThreads), 0, stream, p);
  if (e != cudaSuccess) return e;
  const dim3 blocks(2 * D / 32), threads(32, 32);
  if (p.w_fp32)
    return launch_overlapped(&weight_grad_kernel<float>, blocks, threads, 0, stream, p.partial, ctas, D, static_cast<float*>(dwq),
                             static_cast<float*>(dwk));
  return launch_overlapped(&weight_grad_kernel<T>, blocks, threads, 0, stream, p.partial, ctas, D, static_cast<T*>(dwq),
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
  if (a->axes < 1 || a->axes > 4 || (a->axes > 1 && (a->positions == nullptr || a->pair_axis == nullptr)))
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: 1 to 4 position axes; several need positions and an axis per pair", who);
  if (!(a->eps >= 0.0f) || !std::isfinite(a->eps)) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: eps must be finite and not negative", who);
  if (a->table_rows <= 0 || (a->positions == nullptr && a->table_rows < a->seqlen))
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: the tables must have a row for every position", who);
  for (const long long s : {a->q_batch_stride, a->q_token_stride, a->q_head_stride, a->k_batch_stride, a->k_token_stride,
                            a->k_head_stride})
    if (s % 8 != 0) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: strides must be multiples of 8 elements", who);
  if (backward)
    for (const long long s : {a->dq_batch_stride, a->dq_token_stride, a->dq_head_stride, a->dk_batch_stride, a->dk_token_stride,
                              a->dk_head_stride})
      if (s % 8 != 0) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: strides must be multiples of 8 elements", who);
  p.tokens = static_cast<long long>(a->batch) * a->seqlen;
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
  p.half = a->half;
  p.nope = a->nope;
  p.axes = a->axes;
  p.table_rows = a->table_rows;
  p.w_fp32 = a->weight_dtype == TOKMIX_DTYPE_FP32 ? 1 : 0;
  p.eps = a->eps;
  for (int i = 0; i < a->half; ++i) {
    const int x = a->axes > 1 ? a->pair_axis[i] : 0;
    if (x >= a->axes) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: pair %d names axis %d of %d", who, i, x, a->axes);
    p.axis[i] = static_cast<uint8_t>(x);
  }
  return TOKMIX_OK;
}

void split_units(Params& p, const tokmix_qk_norm_rope* a) {
  p.parts = head_parts(p.tokens, a->heads_q, a->heads_k, a->head_dim);
  p.units = p.tokens * p.parts;
}

}  // namespace qkr
}  // namespace tokmix

extern "C" int tokmix_qk_norm_rope_fwd(const tokmix_qk_norm_rope* a, uint32_t* status, void* stream) {
  using namespace tokmix;
  qkr::Params p{};
  if (const int rc = qkr::prepare("tokmix_qk_norm_rope_fwd", a, false, p)) return rc;
  if (p.tokens == 0) return TOKMIX_OK;
  if (const int rc = check_device()) return rc;
  qkr::split_units(p, a);
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
  const long long units = tokens * qkr::head_parts(tokens, heads_q, heads_k, head_dim);
  return static_cast<long long>(qkr::bwd_ctas(units)) * 2 * head_dim * 4;
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
  qkr::split_units(p, a);
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
