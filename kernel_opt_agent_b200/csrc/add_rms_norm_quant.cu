// add_rms_norm_quant.cu -- residual addition, RMS norm and FP8 quantisation in one pass over a row.
//
// Maths (T = bf16 or fp16, everything else fp32):
//   h = T(x + residual)                        stored: the residual stream of the next layer
//   u = h * weight                             exact in fp32 (8 + 8 or 11 + 11 significant bits)
//   inv_rms = 1 / sqrt(sum h^2 / n + eps)
//   per group of columns:  a = max(max |u|, 2^-100),  y = e4m3(u * (448 / a)),  scale = a * inv_rms / 448
// The row's inv_rms is common to a group and its maximum, so the bytes are formed from u alone: they
// depend on no sum and no order of summation, only the scales carry inv_rms.  2^-100 keeps 448 / a finite
// for a group of zeros (bytes 0).  An infinite or NaN h makes every scale of its row NaN or 0 as the
// formula does.  The scale is formed as a * inv_rms * fp32(1 / 448), at most 2^-24 further off than the division.
//
// Bound: HBM (7 bytes per element against as many flops).  Each row is read once: the CTA's threads hold
// u in fp32 between the sum and the output (rows of more than 32768 columns in 64 registers a thread, so in part in
// local memory: 512 x 65536 96 us, 2.5 TB/s, against 34 us, 6.1 TB/s, for 4096 x 7168; 1024 x 32768 54 us, 4.4 TB/s).
// blockDim = (threads of a row, rows of the CTA).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "host_common.h"

namespace tokmix {
namespace normq {

struct Params {
  const void* x;
  const void* res;  // null: h = x
  const void* w;
  void* res_out;
  uint8_t* y;
  float* scale;
  int rows, n;
  float eps;
};

template <typename T>
__device__ __forceinline__ float2 widen(uint32_t w);
template <>
__device__ __forceinline__ float2 widen<__nv_bfloat16>(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
template <>
__device__ __forceinline__ float2 widen<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t narrow(float a, float b);
template <>
__device__ __forceinline__ uint32_t narrow<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t narrow<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100

// GL lanes of 8 columns make a group (4: 32 columns, 16: 128 columns; 0: the whole row).
template <typename T, int VPT, int GL, int MAXT>
__global__ void __launch_bounds__(MAXT) kernel(const Params p) {
  wait_previous_kernels();
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  const bool act = row < p.rows;
  const int t = threadIdx.x, tpr = blockDim.x;
  const int nvec = p.n >> 3;
  const size_t base = static_cast<size_t>(act ? row : 0) * nvec;
  const uint4* xr = static_cast<const uint4*>(p.x) + base;
  const uint4* rr = static_cast<const uint4*>(p.res) + base;
  uint4* ro = static_cast<uint4*>(p.res_out) + base;

  uint4 x[VPT], r[VPT], wv[VPT];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int i = t + k * tpr;
    const bool in = act && i < nvec;
    x[k] = in ? __ldcs(xr + i) : make_uint4(0u, 0u, 0u, 0u);
    r[k] = in && p.res != nullptr ? __ldcs(rr + i) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int k = 0; k < VPT; ++k) wv[k] = t + k * tpr < nvec ? __ldg(static_cast<const uint4*>(p.w) + t + k * tpr) : make_uint4(0u, 0u, 0u, 0u);
  // h, its sum of squares, u = h * weight (kept: forming it again after the sum costs more than the registers), and the
  // largest |u| of each vector's group
  float ss = 0.0f, amax[VPT], u[VPT][8];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int i = t + k * tpr;
    uint32_t* hw = reinterpret_cast<uint32_t*>(&x[k]);
    if (p.res != nullptr) {
      const uint32_t* rw = reinterpret_cast<const uint32_t*>(&r[k]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = widen<T>(hw[j]), b = widen<T>(rw[j]);
        hw[j] = narrow<T>(a.x + b.x, a.y + b.y);
      }
      if (act && i < nvec) __stcs(ro + i, x[k]);
    }
    const uint32_t* ww = reinterpret_cast<const uint32_t*>(&wv[k]);
    amax[k] = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = widen<T>(hw[j]), w = widen<T>(ww[j]);
      ss += a.x * a.x;
      ss += a.y * a.y;
      u[k][2 * j] = a.x * w.x;
      u[k][2 * j + 1] = a.y * w.y;
      amax[k] = fmaxf(amax[k], fmaxf(fabsf(u[k][2 * j]), fabsf(u[k][2 * j + 1])));
    }
#pragma unroll
    for (int off = GL / 2; off > 0; off >>= 1) amax[k] = fmaxf(amax[k], __shfl_xor_sync(0xffffffffu, amax[k], off));
  }
  float top = 0.0f;  // GL == 0: the row's maximum
  if constexpr (GL == 0) {
#pragma unroll
    for (int k = 0; k < VPT; ++k) top = fmaxf(top, amax[k]);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, off);
    if constexpr (GL == 0) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  }
  if (tpr > 32) {  // rows of several warps (uniform over the CTA)
    __shared__ float part[32], part_top[32];
    const int nw = tpr >> 5, wr = threadIdx.y * nw;
    if ((t & 31) == 0) {
      part[wr + (t >> 5)] = ss;
      part_top[wr + (t >> 5)] = top;
    }
    __syncthreads();
    ss = 0.0f;
    for (int w = 0; w < nw; ++w) {  // the same order for every thread
      ss += part[wr + w];
      if constexpr (GL == 0) top = fmaxf(top, part_top[wr + w]);
    }
  }
  const float inv_rms = 1.0f / sqrtf(ss / static_cast<float>(p.n) + p.eps);
  if (!act) return;
  uint2* yr = reinterpret_cast<uint2*>(p.y) + base;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int i = t + k * tpr;
    if (i >= nvec) break;
    const float a = fmaxf(GL == 0 ? top : amax[k], kTiny);
    const float mul = __fdiv_rn(448.0f, a);
    uint32_t q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      q[j] = __nv_cvt_float2_to_fp8x2(make_float2(u[k][2 * j] * mul, u[k][2 * j + 1] * mul), __NV_SATFINITE, __NV_E4M3);
    __stcs(yr + i, make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16)));
    const float s = a * inv_rms * (1.0f / 448.0f);
    if constexpr (GL == 0) {
      if (i == 0) p.scale[row] = s;
    } else {
      if (i % GL == 0) p.scale[static_cast<size_t>(i / GL) * p.rows + row] = s;
    }
  }
}

template <typename T, int GL>
void launch(const Params& p, cudaStream_t s) {
  const int nvec = p.n / 8;
  // Threads of a row: whole warps with vpt vectors each, few and full (4096 rows of 7168: 4 vectors 34.3 us, 2 44 us,
  // 8 63 us); several short rows share a CTA.
  const int vpt = nvec <= 128 ? 1 : nvec <= 512 ? 2 : nvec <= 2048 ? 4 : 8;
  const int tpr = ((nvec + vpt - 1) / vpt + 31) / 32 * 32;
  const int per = std::max(1, 256 / tpr);
  const dim3 block(static_cast<unsigned>(tpr), static_cast<unsigned>(per));
  const unsigned grid = static_cast<unsigned>((p.rows + per - 1) / per);
  if (vpt == 1)
    launch_overlapped(kernel<T, 1, GL, 256>, grid, block, 0, s, p);
  else if (vpt == 2)
    launch_overlapped(kernel<T, 2, GL, 256>, grid, block, 0, s, p);
  else if (nvec <= 1024)
    launch_overlapped(kernel<T, 4, GL, 256>, grid, block, 0, s, p);
  else if (nvec <= 2048)
    launch_overlapped(kernel<T, 4, GL, 512>, grid, block, 0, s, p);
  else if (nvec <= 4096)
    launch_overlapped(kernel<T, 8, GL, 512>, grid, block, 0, s, p);
  else
    launch_overlapped(kernel<T, 8, GL, 1024>, grid, block, 0, s, p);
}

template <typename T>
void dispatch(const Params& p, int group, cudaStream_t s) {
  if (group == 0)
    launch<T, 0>(p, s);
  else if (group == 32)
    launch<T, 4>(p, s);
  else
    launch<T, 16>(p, s);
}

}  // namespace normq
}  // namespace tokmix

extern "C" int tokmix_add_rms_norm_quant(const void* x, const void* residual, const void* weight, void* residual_out,
                                         void* y_fp8, float* y_scale, int rows, int n, int group, int dtype, float eps,
                                         void* stream) {
  using namespace tokmix;
  using namespace tokmix::normq;
  const char* who = "tokmix_add_rms_norm_quant";
  if (rows < 0 || n <= 0) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: bad shape (%d, %d)", who, rows, n);
  if (group != 0 && group != 32 && group != 128)
    return fail(TOKMIX_ERR_UNSUPPORTED, "%s: group must be 32, 128 or 0 (the row), got %d", who, group);
  if (n % (group ? group : 8) != 0 || n > 65536)
    return fail(TOKMIX_ERR_UNSUPPORTED, "%s: row length must be a multiple of %d and at most 65536 (got %d)", who,
                group ? group : 8, n);
  if (dtype != TOKMIX_DTYPE_BF16 && dtype != TOKMIX_DTYPE_FP16)
    return fail(TOKMIX_ERR_UNSUPPORTED, "%s: bf16 or fp16 only (dtype %d)", who, dtype);
  if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: bad eps", who);
  if (rows > 0x7fffff00) return fail(TOKMIX_ERR_UNSUPPORTED, "%s: at most 2^31 - 256 rows (got %d)", who, rows);  // int row indexes
  if (rows == 0) return TOKMIX_OK;
  if (!x || !weight || !y_fp8 || !y_scale || (residual && !residual_out))
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: null pointer argument", who);
  for (const void* ptr : {x, residual, weight, static_cast<const void*>(residual_out), static_cast<const void*>(y_fp8)})
    if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0)
      return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: tensors must be 16-byte aligned", who);
  if (const int rc = check_device()) return rc;
  Params p{x, residual, weight, residual_out, static_cast<uint8_t*>(y_fp8), y_scale, rows, n, eps};
  if (dtype == TOKMIX_DTYPE_BF16)
    dispatch<__nv_bfloat16>(p, group, static_cast<cudaStream_t>(stream));
  else
    dispatch<__half>(p, group, static_cast<cudaStream_t>(stream));
  return check_launch(who);
}
