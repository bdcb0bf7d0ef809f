// kv8_append.cu -- new keys and values enter the paged 8-bit cache.
//
// Maths, per (page, head), for keys and for values apart.  Let the page hold tokens x_t.  Its scale is
//   s = 2^e,  e = the smallest integer >= -100 with max_t |x_t| <= qmax 2^e   (qmax 448 e4m3, 127 int8)
// and a value is held as round(x / s).  When new tokens arrive on a page that already holds some,
//   s' = max(s, scale of the new tokens),   old bytes q -> round(q s / s')   if s' > s.
// Powers of two make x / s exact, so each rounding is the type's own; rounding an e4m3 value again after
// the scale grew changes only values that fall among e4m3's subnormals, and an int8 value is off by at
// most one step of the final scale however often it was rounded (1/2 + 1/4 + ... steps).  Appending at
// the same positions again gives the same bytes.
//
// Bound: HBM.  2 bytes read and 1 written per value; a page's tokens are read once, held in registers for
// the maximum, and written.  One unit = (sequence, page the call touches, head, key or value): the page
// is in one unit's hands, so no atomics and no order between units.  A unit of few vectors (a decode
// step: one row) takes a warp, a unit of up to a whole page a CTA of 256 threads.
#include "kv8_common.cuh"

#include <algorithm>

namespace tokmix {
namespace kv8 {

struct AppendParams {
  View c;
  const void* k;
  const void* v;
  long long k_sb, k_st, k_sh, v_sb, v_st, v_sh;  // element strides of the new keys and values
  int rows;          // new tokens per sequence at most
  uint32_t touched;  // pages a sequence can touch
  int d, d_shift;
  uint32_t units;
  uint32_t* status;
};

// scale of a page whose largest magnitude is a (finite)
template <bool E4M3>
__device__ __forceinline__ float pow2_scale(float a) {
  const uint32_t bits = __float_as_uint(a);
  const int ex = static_cast<int>(bits >> 23);
  const uint32_t man = bits & 0x7fffffu;
  // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
  const int e = E4M3 ? ex - 135 + (man > 0x600000u) : ex - 133 + (man > 0x7e0000u);
  return __uint_as_float(static_cast<uint32_t>(max(e, -100) + 127) << 23);
}

template <typename T>
struct Half16;
template <>
struct Half16<__nv_bfloat16> {
  static constexpr uint32_t kInf = 0x7f80u;
  // larger magnitude of each half (its sign is of no use), NaN if either is
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m = __hmax2_nan(__habs2(*reinterpret_cast<const __nv_bfloat162*>(&a)), __habs2(*reinterpret_cast<const __nv_bfloat162*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  static __device__ __forceinline__ float widen(uint32_t b) { return __uint_as_float(b << 16); }
  static __device__ __forceinline__ float2 widen2(uint32_t w) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
  }
};
template <>
struct Half16<__half> {
  static constexpr uint32_t kInf = 0x7c00u;
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2_nan(__habs2(*reinterpret_cast<const __half2*>(&a)), __habs2(*reinterpret_cast<const __half2*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  static __device__ __forceinline__ float widen(uint32_t b) { return __half2float(__ushort_as_half(static_cast<uint16_t>(b))); }
  static __device__ __forceinline__ float2 widen2(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
};

// GT threads work on a unit (a warp: eight units per CTA; more: one), NV vectors of 8 values each.
template <typename T, bool E4M3, int NV, int GT>
__global__ void __launch_bounds__(GT == 32 ? 256 : GT) append_kernel(const AppendParams p) {
  constexpr int kUnits = GT == 32 ? 8 : 1;
  wait_previous_kernels();
  const View& c = p.c;
  const uint32_t unit = blockIdx.x * kUnits + threadIdx.x / GT;
  if (unit >= p.units) return;  // warp-uniform (a warp per unit), never (a CTA per unit)
  const int lane = threadIdx.x & (GT - 1);
  const bool is_v = (unit & 1) != 0;
  const uint32_t page_of = (unit >> 1) / p.c.hkv;  // 32-bit divisions: 64-bit ones cost more than the page's values do
  const int h = static_cast<int>((unit >> 1) - page_of * p.c.hkv);
  const int b = static_cast<int>(page_of / p.touched);
  const int j = static_cast<int>(page_of - b * p.touched);

  const Seq s = load_seq(c, b, p.rows);
  if (!s.ok) {
    if (lane == 0) report_bad(p.status);
    return;
  }
  const int pj = (s.start >> c.page_shift) + j;
  const int page0 = pj << c.page_shift;  // position of the page's first slot
  const int lo = max(s.start, page0), hi = min(s.end, page0 + c.page);
  if (lo >= hi) return;  // a page the sequence does not reach
  const int pid = __ldg(c.table + static_cast<long long>(b) * c.table_stride + pj);  // used behind the tokens' loads
  const T* src = is_v ? static_cast<const T*>(p.v) + b * p.v_sb + h * p.v_sh : static_cast<const T*>(p.k) + b * p.k_sb + h * p.k_sh;
  const long long st = is_v ? p.v_st : p.k_st;
  src += (lo - s.start) * st;

  const int vshift = p.d_shift - 3;  // vectors per token: 1 << vshift
  const int nvec = (hi - lo) << vshift;
  uint4 x[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int vi = lane + i * GT;
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    if (vi < nvec) x[i] = __ldcs(reinterpret_cast<const uint4*>(src + (vi >> vshift) * st) + (vi & ((1 << vshift) - 1)));
  }
  if (pid < 0 || pid >= c.num_pages) {
    if (lane == 0) report_bad(p.status);
    return;  // the whole unit
  }
  uint8_t* tile = is_v ? c.v + pid * c.v_page_stride + h * c.v_head_stride : c.k + pid * c.k_page_stride + h * c.k_head_stride;
  float* scale = (is_v ? c.v_scale : c.k_scale) + static_cast<long long>(pid) * c.hkv + h;
  const bool has_old = lo > page0;
  const float s_old = has_old ? *scale : 0.0f;

  uint32_t amax2 = 0;  // packed magnitudes; a NaN stays one
#pragma unroll
  for (int i = 0; i < NV; ++i)
    amax2 = Half16<T>::max2(Half16<T>::max2(Half16<T>::max2(amax2, x[i].x), Half16<T>::max2(x[i].y, x[i].z)), x[i].w);
  amax2 &= 0x7fff7fffu;  // as integers, magnitudes order like the values, NaN above infinity
  uint32_t amax = __reduce_max_sync(0xffffffffu, max(amax2 & 0xffffu, amax2 >> 16));
  if constexpr (GT > 32) {
    __shared__ uint32_t part[GT / 32];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
    __syncthreads();  // also: every thread has read the old scale
#pragma unroll
    for (int w = 0; w < GT / 32; ++w) amax = max(amax, part[w]);
  } else {
    __syncwarp();  // every lane has read the old scale
  }
  float s_new = fmaxf(s_old, pow2_scale<E4M3>(Half16<T>::widen(amax)));
  if (amax >= Half16<T>::kInf || isnan(s_old)) {  // the block reads as NaN from here on
    s_new = __uint_as_float(0x7fc00000u);
    // the scale alone marks it: a NaN byte would reach rows that do not see it (0 * NaN)
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  if (lane == 0) *scale = s_new;

  const float inv = isnan(s_new) ? 0.0f : 1.0f / s_new;  // exact
  uint8_t* dst = tile + ((lo - page0) << p.d_shift);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int vi = lane + i * GT;
    if (vi < nvec) {
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      float f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 t = Half16<T>::widen2(w[e]);
        f[2 * e] = t.x * inv;
        f[2 * e + 1] = t.y * inv;
      }
      *reinterpret_cast<uint2*>(dst + (static_cast<size_t>(vi) << 3)) =
          make_uint2(float4_to_bytes<E4M3>(f[0], f[1], f[2], f[3]), float4_to_bytes<E4M3>(f[4], f[5], f[6], f[7]));
    }
  }
  if (has_old && s_old < s_new) {  // (false for a NaN scale)
    const float ratio = s_old / s_new;
    const int n16 = (lo - page0) << (p.d_shift - 4);
    for (int i = lane; i < n16; i += GT) {
      uint4 q = reinterpret_cast<uint4*>(tile)[i];
      uint32_t* w = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f[4];
        bytes_to_float4<E4M3>(w[e], f);
        w[e] = float4_to_bytes<E4M3>(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
      }
      reinterpret_cast<uint4*>(tile)[i] = q;
    }
  }
}

template <typename T, bool E4M3>
void launch_append(const AppendParams& p, cudaStream_t s) {
  const int most = std::min(p.rows, p.c.page) << (p.d_shift - 3);  // vectors of the largest unit
  // 8 vectors a thread keep enough loads in flight and few enough threads busy with the unit's pointers (4 prompts of
  // 8192 tokens, Hkv 8, D 128, pages of 64: 128 threads x 8 23.4 us, 256 x 4 30.2 us, 64 x 16 28.5 us)
  if (most <= 4 * 32)
    launch_overlapped(append_kernel<T, E4M3, 4, 32>, dim3((p.units + 7) / 8), dim3(256), 0, s, p);
  else if (most <= 8 * 128)
    launch_overlapped(append_kernel<T, E4M3, 8, 128>, dim3(p.units), dim3(128), 0, s, p);
  else if (most <= 8 * 256)
    launch_overlapped(append_kernel<T, E4M3, 8, 256>, dim3(p.units), dim3(256), 0, s, p);
  else
    launch_overlapped(append_kernel<T, E4M3, 16, 256>, dim3(p.units), dim3(256), 0, s, p);
}

int make_view(const char* who, const tokmix_kv8_cache* c, View& out) {
  if (c == nullptr) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: null cache", who);
  if (c->dtype != TOKMIX_DTYPE_E4M3 && c->dtype != TOKMIX_DTYPE_INT8)
    return fail(TOKMIX_ERR_UNSUPPORTED, "%s: the cache holds e4m3 or int8 (dtype %d)", who, c->dtype);
  if (c->batch < 0 || c->num_pages <= 0 || c->heads_kv <= 0 || c->max_pages < 0)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: bad cache sizes", who);
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return fail(TOKMIX_ERR_UNSUPPORTED, "%s: page_size must be 16, 32, 64 or 128 (got %d)", who, c->page_size);
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(TOKMIX_ERR_UNSUPPORTED, "%s: head_dim must be 64, 128 or 256 (got %d)", who, c->head_dim);
  if (static_cast<long long>(c->max_pages) * c->page_size > 0x7fffffffLL - 4096)
    return fail(TOKMIX_ERR_UNSUPPORTED, "%s: more than 2^31 positions per sequence", who);
  const long long tile = static_cast<long long>(c->page_size) * c->head_dim;
  for (const long long st : {c->k_page_stride, c->k_head_stride, c->v_page_stride, c->v_head_stride})
    if (st % 16 != 0 || st < tile)
      return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: page and head strides must be multiples of 16 and at least a tile", who);
  if (c->k_page_stride > 0xffffffffLL || c->v_page_stride > 0xffffffffLL)
    return fail(TOKMIX_ERR_UNSUPPORTED, "%s: pages more than 4 GB apart", who);
  if (c->table_stride < c->max_pages) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: bad table stride", who);
  if (c->batch > 0) {
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->seq_lens || (c->max_pages > 0 && !c->block_table))
      return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: null pointer in the cache", who);
    if (reinterpret_cast<uintptr_t>(c->k) % 16 != 0 || reinterpret_cast<uintptr_t>(c->v) % 16 != 0)
      return fail(TOKMIX_ERR_INVALID_ARGUMENT, "%s: the cache must be 16-byte aligned", who);
  }
  out.k = static_cast<uint8_t*>(c->k);
  out.v = static_cast<uint8_t*>(c->v);
  out.k_scale = c->k_scale;
  out.v_scale = c->v_scale;
  out.k_page_stride = c->k_page_stride;
  out.k_head_stride = c->k_head_stride;
  out.v_page_stride = c->v_page_stride;
  out.v_head_stride = c->v_head_stride;
  out.table = c->block_table;
  out.table_stride = c->table_stride;
  out.seq_lens = c->seq_lens;
  out.new_lens = c->new_lens;
  out.num_pages = c->num_pages;
  out.page = c->page_size;
  out.page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  out.hkv = c->heads_kv;
  out.batch = c->batch;
  out.max_pages = c->max_pages;
  return TOKMIX_OK;
}

}  // namespace kv8
}  // namespace tokmix

extern "C" int tokmix_kv8_append(const void* k, long long k_batch_stride, long long k_token_stride,
                                 long long k_head_stride, const void* v, long long v_batch_stride,
                                 long long v_token_stride, long long v_head_stride, int tokens, int io_dtype,
                                 const tokmix_kv8_cache* cache, uint32_t* status, void* stream) {
  using namespace tokmix;
  using namespace tokmix::kv8;
  AppendParams p{};
  if (const int rc = make_view("tokmix_kv8_append", cache, p.c)) return rc;
  if (tokens < 0) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_kv8_append: negative token count");
  if (io_dtype != TOKMIX_DTYPE_BF16 && io_dtype != TOKMIX_DTYPE_FP16)
    return fail(TOKMIX_ERR_UNSUPPORTED, "tokmix_kv8_append: new keys and values are bf16 or fp16 (dtype %d)", io_dtype);
  if (tokens == 0 || p.c.batch == 0) return TOKMIX_OK;
  if (!k || !v) return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_kv8_append: null pointer argument");
  if (reinterpret_cast<uintptr_t>(k) % 16 != 0 || reinterpret_cast<uintptr_t>(v) % 16 != 0)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_kv8_append: k and v must be 16-byte aligned");
  for (const long long st : {k_batch_stride, k_token_stride, k_head_stride, v_batch_stride, v_token_stride, v_head_stride})
    if (st % 8 != 0 || st < 0)
      return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_kv8_append: strides of k and v must be multiples of 8 elements");
  // a key's unit and a value's would race for the same tile and scale
  if (cache->k == cache->v || cache->k_scale == cache->v_scale)
    return fail(TOKMIX_ERR_INVALID_ARGUMENT, "tokmix_kv8_append: keys and values need a cache and scales each");
  p.k = k;
  p.v = v;
  p.k_sb = k_batch_stride;
  p.k_st = k_token_stride;
  p.k_sh = k_head_stride;
  p.v_sb = v_batch_stride;
  p.v_st = v_token_stride;
  p.v_sh = v_head_stride;
  p.rows = tokens;
  p.touched = (tokens + p.c.page - 2) / p.c.page + 1;  // one token: 1; a page may be entered at any slot
  p.d = cache->head_dim;
  p.d_shift = p.d == 64 ? 6 : p.d == 128 ? 7 : 8;
  const long long units = 2LL * p.c.batch * p.touched * p.c.hkv;
  if (units > 0x7FFFFFFFLL) return fail(TOKMIX_ERR_UNSUPPORTED, "tokmix_kv8_append: problem too large");
  p.units = static_cast<uint32_t>(units);
  p.status = status;
  if (const int rc = check_device()) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool e4m3 = cache->dtype == TOKMIX_DTYPE_E4M3;
  if (io_dtype == TOKMIX_DTYPE_BF16)
    e4m3 ? launch_append<__nv_bfloat16, true>(p, s) : launch_append<__nv_bfloat16, false>(p, s);
  else
    e4m3 ? launch_append<__half, true>(p, s) : launch_append<__half, false>(p, s);
  return check_launch("tokmix_kv8_append");
}
