// kv4_attn.cu -- grouped-query attention over the 4-bit KV cache.
//
// out = softmax(q K^T / sqrt(128)) V for every new token of every sequence, K
// and V the values m + d c the cache rows stand for (the fp16 cache's
// counterpart is mlm_attn_decode; LlamaRunner.swift:669-952).
//
// One warp per (sequence, token, query head) walks the rows the token sees with
// a running maximum and sum; a lane holds dimensions 4l .. 4l+3.
#include <algorithm>

#include "mlm_device.cuh"
#include "mlm_internal.h"

namespace mlm {
namespace {

constexpr int kRow = MLM_KV4_ROW_BYTES;
constexpr int kD = 128;

// the lane's four values of a cache row
__device__ __forceinline__ float4 row4(const uint8_t *row, int lane) {
  const uint32_t w = *reinterpret_cast<const uint16_t *>(row + 2 * lane);
  const float2 dm = __half22float2(*reinterpret_cast<const __half2 *>(row + 64 + 4 * (lane / 8)));
  return make_float4(fmaf(dm.x, (float)(w & 15u), dm.y), fmaf(dm.x, (float)((w >> 4) & 15u), dm.y),
                     fmaf(dm.x, (float)((w >> 8) & 15u), dm.y), fmaf(dm.x, (float)(w >> 12), dm.y));
}

template <class OutT>
__global__ void __launch_bounds__(128) kv4_attn_simple_kernel(
    const uint8_t *kc, const uint8_t *vc, const __half *q, OutT *out, int batch, int tokens,
    int n_heads, int n_kv, int capacity, const int32_t *lens, const int32_t *counts, int *status) {
  pdl_wait_then_release();
  const long long i = (long long)blockIdx.x * 4 + threadIdx.x / 32;
  const int lane = threadIdx.x & 31;
  if (i >= (long long)batch * tokens * n_heads) return;
  const int head = (int)(i % n_heads);
  const int t = (int)(i / n_heads % tokens);
  const int b = (int)(i / n_heads / tokens);
  int len = lens[b], count = counts ? counts[b] : tokens;
  if (len < 0 || len > capacity || count < 0 || count > tokens) {
    if (lane == 0) *status = MLM_ERR_SHAPE;
    len = min(max(len, 0), capacity);
    count = min(max(count, 0), tokens);
  }
  if (t >= count) return;
  const int seen = max(0, len - count + t + 1);
  const size_t at = (size_t)i * kD + 4 * lane;
  float x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = __half2float(q[at + e]);
  const size_t row0 = ((size_t)b * n_kv + head / (n_heads / n_kv)) * capacity;
  float top = -INFINITY, sum = 0.f, o[4] = {};
  for (int j = 0; j < seen; ++j) {
    const float4 k = row4(kc + (row0 + j) * kRow, lane);
    const float s = warp_sum(x[0] * k.x + x[1] * k.y + x[2] * k.z + x[3] * k.w) * 0.08838834764831845f;
    const float up = fmaxf(top, s);
    const float old = top == up ? 1.f : expf(top - up), p = expf(s - up);
    const float4 v = row4(vc + (row0 + j) * kRow, lane);
    o[0] = o[0] * old + p * v.x;
    o[1] = o[1] * old + p * v.y;
    o[2] = o[2] * old + p * v.z;
    o[3] = o[3] * old + p * v.w;
    sum = sum * old + p;
    top = up;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) out[at + e] = from_float<OutT>(seen ? o[e] / sum : 0.f);
}

template <class OutT>
int simple(mlm_ctx *ctx, const mlm_kv4_cache &c, const void *q, int n_heads, int tokens,
           const int32_t *lens, const int32_t *counts, void *out) {
  const long long warps = (long long)c.batch * tokens * n_heads;
  return check_launch_pdl(
      ctx,
      launch_pdl(kv4_attn_simple_kernel<OutT>, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0,
                 ctx->stream, reinterpret_cast<const uint8_t *>(c.k),
                 reinterpret_cast<const uint8_t *>(c.v), reinterpret_cast<const __half *>(q),
                 reinterpret_cast<OutT *>(out), c.batch, tokens, n_heads, c.n_kv_heads, c.capacity,
                 lens, counts, ctx->dev_status),
      "mlm_attn_kv4");
}

}  // namespace

int kv4_attn_init(mlm_ctx *) { return MLM_OK; }

}  // namespace mlm

using namespace mlm;

extern "C" int mlm_attn_kv4(mlm_ctx *ctx, const mlm_kv4_cache *cache, const void *q, int n_heads,
                            int tokens, const int32_t *lens, const int32_t *counts, void *out,
                            int out_type) {
  MLM_CHECK_CTX(ctx);
  const int st = kv4_check(ctx, cache, "mlm_attn_kv4");
  if (st != MLM_OK) return st;
  MLM_REQUIRE(ctx, q && out && lens, MLM_ERR_ARG, "mlm_attn_kv4: null buffer");
  MLM_REQUIRE(ctx, aligned16(q) && aligned16(out) && aligned4(lens) && aligned4(counts),
              MLM_ERR_ALIGN,
              "mlm_attn_kv4: q and out must be 16-byte, lengths and counts 4-byte aligned");
  MLM_REQUIRE(ctx, out_type == MLM_TYPE_F16 || out_type == MLM_TYPE_BF16, MLM_ERR_UNSUPPORTED,
              "mlm_attn_kv4: output type %d (F16 %d or BF16 %d)", out_type, MLM_TYPE_F16,
              MLM_TYPE_BF16);
  MLM_REQUIRE(ctx, n_heads > 0 && n_heads <= 16384 && n_heads % cache->n_kv_heads == 0,
              MLM_ERR_SHAPE, "mlm_attn_kv4: %d query heads not a multiple of %d KV heads", n_heads,
              cache->n_kv_heads);
  MLM_REQUIRE(ctx, tokens > 0 && tokens <= 65536, MLM_ERR_SHAPE,
              "mlm_attn_kv4: tokens=%d (1 .. 65536)", tokens);
  DeviceGuard guard(ctx);
  if (out_type == MLM_TYPE_F16)
    return simple<__half>(ctx, *cache, q, n_heads, tokens, lens, counts, out);
  return simple<__nv_bfloat16>(ctx, *cache, q, n_heads, tokens, lens, counts, out);
}
