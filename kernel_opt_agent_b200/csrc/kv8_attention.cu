// kv8_attention.cu -- attention of a few new tokens per sequence over the paged 8-bit cache.
//
//   o = softmax(q k^T * sm_scale) v,   k, v = byte * scale of the token's (page, head)
//
// One CTA per (sequence, query token, query head); four warps share the tokens, a lane holds head_dim / 32
// elements of the query and the output.  Running maximum and sum per warp in fp32, joined at the end.
#include "kv8_common.cuh"

#include <cmath>

namespace tokmix {
namespace kv8 {

constexpr int kMaxTokens = 16;

struct AttnParams {
  View c;
  const void* q;
  long long q_sb, q_st, q_sh;
  void* out;
  float* lse;
  int tokens, hq;
  int bf16;
  float scale_log2;  // sm_scale * log2(e)
  uint32_t* status;
};

template <int D, bool E4M3>
__global__ void __launch_bounds__(128) attn_simple_kernel(const AttnParams p) {
  constexpr int E = D / 32;
  const View& c = p.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.x % p.hq;
  const int rest = blockIdx.x / p.hq;
  const int i = rest % p.tokens, b = rest / p.tokens;
  const int kvh = h / (p.hq / c.hkv);
  const Seq s = load_seq(c, b, p.tokens);
  const int lim = i < s.end - s.start ? s.start + i + 1 : 0;
  if (!s.ok && threadIdx.x == 0) report_bad(p.status);

  float q[E], acc[E];
  const long long qo = b * p.q_sb + i * p.q_st + h * p.q_sh;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const long long at = qo + lane * E + e;
    q[e] = p.bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.q)[at]) : __half2float(static_cast<const __half*>(p.q)[at]);
    acc[e] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int t = warp; t < lim; t += 4) {
    const int pid = __ldg(c.table + b * c.table_stride + (t >> c.page_shift));
    const bool bad = pid < 0 || pid >= c.num_pages;
    const long long pg = bad ? 0 : pid;
    if (bad && lane == 0) report_bad(p.status);
    const float nan = __uint_as_float(0x7fc00000u);
    const float ks = bad ? nan : c.k_scale[pg * c.hkv + kvh], vs = bad ? nan : c.v_scale[pg * c.hkv + kvh];
    const int slot = t & (c.page - 1);
    const uint8_t* kp = c.k + pg * c.k_page_stride + kvh * c.k_head_stride + slot * D + lane * E;
    const uint8_t* vp = c.v + pg * c.v_page_stride + kvh * c.v_head_stride + slot * D + lane * E;
    float dot = 0.0f, v[E];
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      float f[4], g[4];
      bytes_to_float4<E4M3>(*reinterpret_cast<const uint16_t*>(kp + e), f);
      bytes_to_float4<E4M3>(*reinterpret_cast<const uint16_t*>(vp + e), g);
      dot += q[e] * f[0] + q[e + 1] * f[1];
      v[e] = g[0];
      v[e + 1] = g[1];
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    const float sc = dot * ks * p.scale_log2;
    const float m_new = fmaxf(m, sc);
    const float ref = m_new == -INFINITY ? 0.0f : m_new;
    const float corr = exp2f(m - ref), w = exp2f(sc - ref);
    l = l * corr + w;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * corr + w * vs * v[e];
    m = m_new;
  }
  __shared__ float sm_m[4], sm_l[4], sm_o[4][D];
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) sm_o[warp][lane * E + e] = acc[e];
  __syncthreads();
  float top = -INFINITY, sum = 0.0f, w[4];
  for (int x = 0; x < 4; ++x) top = fmaxf(top, sm_m[x]);
  const float ref = top == -INFINITY ? 0.0f : top;
  for (int x = 0; x < 4; ++x) {
    w[x] = exp2f(sm_m[x] - ref);
    sum += w[x] * sm_l[x];
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const size_t row = static_cast<size_t>(blockIdx.x);
  for (int e = threadIdx.x; e < D; e += 128) {
    float o = 0.0f;
    for (int x = 0; x < 4; ++x) o += w[x] * sm_o[x][e];
    o *= inv;
    if (!s.ok) o = __uint_as_float(0x7fc00000u);
    if (p.bf16)
      static_cast<__nv_bfloat16*>(p.out)[row * D + e] = __float2bfloat16_rn(o);
    else
      static_cast<__half*>(p.out)[row * D + e] = __float2half_rn(o);
  }
  if (p.lse != nullptr && threadIdx.x == 0)
    p.lse[row] = !s.ok ? __uint_as_float(0x7fc00000u) : sum == 0.0f ? -INFINITY : (ref + log2f(sum)) * 0.6931471805599453f;
}

template <int D>
void launch_attn(const AttnParams& p, bool e4m3, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(p.c.batch) * p.tokens * p.hq;
  if (e4m3)
    attn_simple_kernel<D, true><<<grid, 128, 0, s>>>(p);
  else
    attn_simple_kernel<D, false><<<grid, 128, 0, s>>>(p);
}

}  // namespace kv8
}  // namespace tokmix

extern "C" long long tokmix_kv8_attention_workspace_bytes(int tokens, int heads_q, int heads_kv, int head_dim) {
  using namespace tokmix::kv8;
  if (tokens < 1 || tokens > kMaxTokens || heads_kv <= 0 || heads_q <= 0 || heads_q % heads_kv != 0 ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return -1;
  return 16;
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
  if (static_cast<long long>(p.c.batch) * tokens * heads_q > 0x7fffffffLL)
    return fail(TOKMIX_ERR_UNSUPPORTED, "%s: problem too large", who);
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
  p.bf16 = io_dtype == TOKMIX_DTYPE_BF16;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool e4m3 = cache->dtype == TOKMIX_DTYPE_E4M3;
  if (cache->head_dim == 64)
    launch_attn<64>(p, e4m3, s);
  else if (cache->head_dim == 128)
    launch_attn<128>(p, e4m3, s);
  else
    launch_attn<256>(p, e4m3, s);
  return check_launch(who);
}
