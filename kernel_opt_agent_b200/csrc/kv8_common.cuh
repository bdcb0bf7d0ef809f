// kv8_common.cuh -- what the kernels over the paged 8-bit key/value cache share: the cache's device
// view, the per-sequence lengths with their checks, and the conversions between a cached byte and
// the value it stands for.
//
// A cache holds pages of `page` tokens: bytes [num_pages][heads_kv][page][head_dim] (e4m3 or int8; the
// page and head strides are free, a (page, head) tile is contiguous) and one fp32 scale per (page,
// head) for keys and one for values.  A cached value is byte * scale.  Scales written by
// tokmix_kv8_append are powers of two, so that multiplication is exact and the value of a byte is
// exactly representable in bf16.  A NaN scale marks a block that was given a value that is not
// finite: all of it reads as NaN.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "host_common.h"

namespace tokmix {
namespace kv8 {

constexpr uint32_t kStatusBadArgs = TOKMIX_DEV_BAD_ARGS;

struct View {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;  // [num_pages, hkv]
  float* v_scale;
  long long k_page_stride, k_head_stride, v_page_stride, v_head_stride;  // bytes (= elements)
  const int32_t* table;  // [batch, max_pages], rows table_stride apart
  long long table_stride;
  const int32_t* seq_lens;  // [batch] tokens in the cache, the newest included
  const int32_t* new_lens;  // [batch] or null (every row of the call)
  int num_pages, page, page_shift, hkv, batch, max_pages;
};

// Checks a cache description on the host and makes the device view; head_dim is returned for dispatch.
int make_view(const char* who, const tokmix_kv8_cache* c, View& out);

// Sets the bit and keeps the word's others.  The word may be device memory or mapped host memory (where the operation is atomic
// for this device's kernels, not towards the host).
__device__ __forceinline__ void report_bad(uint32_t* status) {
  if (status != nullptr) atomicOr(status, kStatusBadArgs);
}

struct Seq {
  int start;  // position of the first new token
  int end;    // tokens in the cache (position after the last)
  bool ok;    // the lengths fit the call and the table
};

// Lengths of sequence b in a call with `rows` new tokens per sequence.
__device__ __forceinline__ Seq load_seq(const View& c, int b, int rows) {
  const int end = __ldg(c.seq_lens + b);
  const int n = c.new_lens != nullptr ? __ldg(c.new_lens + b) : rows;
  Seq s;
  s.ok = n >= 0 && n <= rows && end >= n && static_cast<long long>(end) <= static_cast<long long>(c.max_pages) * c.page;
  s.end = s.ok ? end : 0;
  s.start = s.ok ? end - n : 0;
  return s;
}

// Two e4m3 bytes (low byte first) -> two halves; exact.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint16_t b) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(b, __NV_E4M3);
  return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
}

// Four cached bytes -> four floats (before the scale); exact.
template <bool E4M3>
__device__ __forceinline__ void bytes_to_float4(uint32_t w, float (&f)[4]) {
  if constexpr (E4M3) {
    const uint32_t a = e4m3x2_to_half2(static_cast<uint16_t>(w)), b = e4m3x2_to_half2(static_cast<uint16_t>(w >> 16));
    const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a));
    const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
    f[0] = fa.x;
    f[1] = fa.y;
    f[2] = fb.x;
    f[3] = fb.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
  }
}

// Four floats (already divided by the scale, so within the type's range) -> four bytes, rounded to
// nearest, ties to even.
template <bool E4M3>
__device__ __forceinline__ uint32_t float4_to_bytes(float a, float b, float c, float d) {
  if constexpr (E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  } else {
    const uint32_t x = static_cast<uint32_t>(__float2int_rn(a)) & 0xffu, y = static_cast<uint32_t>(__float2int_rn(b)) & 0xffu;
    const uint32_t z = static_cast<uint32_t>(__float2int_rn(c)) & 0xffu, w = static_cast<uint32_t>(__float2int_rn(d)) & 0xffu;
    return x | (y << 8) | (z << 16) | (w << 24);
  }
}

}  // namespace kv8
}  // namespace tokmix
