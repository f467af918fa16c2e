// kv4.cu -- rows of the 4-bit KV cache: quantizing append and read-back.
//
// A cache row is 80 bytes: 64 bytes of 4-bit codes and four fp16 pairs (d, m),
// one per group of 32 elements, element i standing for m + d c.  The append
// takes K and V rows where the projection left them (fp32, fp16 or bf16, any
// row stride); the reference's counterpart is the fp16 cache blit of
// LlamaRunner.swift:643-666.
//
// Half a warp owns a row: lane l of it holds elements 8l .. 8l+7, so a group's
// minimum and maximum take two shuffles over four lanes and its eight codes
// are one 32-bit word.  Its K and V loads are in flight together; both halves of a
// warp take neighbouring tokens of one head, whose cache rows are neighbours.
// (Two tokens per half warp instead: 1024 fp32 rows x 8 heads appended and read back
// 7.7 us, one 5.4.)  Bound by bytes: a row is read once (512 or 256 B) and 80 B are
// written; 16 ragged prompts of up to 509 fp16 tokens x 8 heads appended and read back,
// 43 MB, take 14.5 us in a graph, one token 3.1 us.
#include <algorithm>

#include "kv4_common.cuh"

// Pointers carry no __restrict__: their data may come from the kernel this one
// is a programmatic dependent of, so no load may move above the dependent wait,
// as the compiler may do with loads it takes for invariant.
namespace mlm {
namespace {

constexpr int kRow = MLM_KV4_ROW_BYTES;
constexpr int kD = 128;
constexpr int kThreads = 256;
constexpr int kRowsPerCta = kThreads / 16;
// inputs are kept within this, so that m + 15 d stays an fp16 value however d
// was rounded (by at most 4, half the spacing of fp16 values above 8192)
constexpr float kLimit = 65408.f;

// minimum and maximum that return NaN when an operand is NaN
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// elements p[0..8) as fp32 (p 16-byte aligned)
__device__ __forceinline__ void load8(const float *p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4 *>(p);
  const float4 b = *(reinterpret_cast<const float4 *>(p) + 1);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
  x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void load8(const __half *p, float (&x)[8]) {
  const uint4 r = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&x)[8]) {
  const uint4 r = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// Eight elements of a row to their code word; the group's (d, m) as fp16 bits.
// The four lanes of a group call this together.  Elements beyond the limit need no
// clamp of their own: the group's bounds are clamped, and such an element's code
// is 0 or 15 as its clamped value's.
__device__ __forceinline__ uint32_t quantize8(const float (&x)[8], uint32_t &dm) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  lo = min_nan(max_nan(lo, -kLimit), kLimit);
  hi = min_nan(max_nan(hi, -kLimit), kLimit);
  const __half m16 = __float2half_rn(lo);
  const float m = __half2float(m16);
  const __half d16 = __float2half_rn(__fmul_rn(__fsub_rn(hi, m), 1.0f / 15.0f));
  const float d = __half2float(d16);
  const float inv = d > 0.f ? __frcp_rn(d) : 0.f;
  dm = (uint32_t)__half_as_ushort(d16) | ((uint32_t)__half_as_ushort(m16) << 16);
  // 1.5 2^23 + c has c in its low bits (rounded half to even); the words' sum of such
  // bits, shifted, is the code word and a constant
  constexpr float kMagic = 12582912.f;
  constexpr uint32_t kMagicBits = 0x4B400000u;
  uint32_t word = 0, bias = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = fminf(fmaxf(__fmul_rn(__fsub_rn(x[i], m), inv), 0.f), 15.f);  // NaN: 0
    word += __float_as_uint(__fadd_rn(c, kMagic)) << (4 * i);
    bias += kMagicBits << (4 * i);
  }
  return word - bias;
}

// Where half a warp's row lies; false where there is none.  A grid row per sequence,
// rows head first, token second: 32-bit indexes, one division.
struct RowAt {
  size_t source_row;  // among [batch][tokens]
  int h;
  size_t cache_row;
};
__device__ __forceinline__ bool row_at(int n_kv, int tokens, int capacity, const int32_t *pos,
                                       const int32_t *counts, int *status, RowAt &r) {
  const uint32_t i = blockIdx.x * kRowsPerCta + threadIdx.x / 16;
  const int b = blockIdx.y;
  r.h = (int)(i / (uint32_t)tokens);
  if (r.h >= n_kv) return false;
  const int t = (int)(i - (uint32_t)r.h * (uint32_t)tokens);
  const bool report = r.h == 0 && (threadIdx.x & 15) == 0;  // one lane of the row
  const int first = pos[b];
  if (counts) {
    const int n = counts[b];
    if ((n < 0 || n > tokens) && t == 0 && report) report_outside(status);
    if (t >= n) return false;
  }
  const long long slot = (long long)first + t;
  if (slot < 0 || slot >= capacity) {
    if (report) report_outside(status);
    return false;
  }
  r.source_row = (size_t)b * tokens + t;
  r.cache_row = ((size_t)b * n_kv + r.h) * capacity + (size_t)slot;
  return true;
}

template <class T>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(
    const T *k, const T *v, long long row_stride, int n_kv, int tokens, int capacity,
    const int32_t *pos, const int32_t *counts, uint8_t *kc, uint8_t *vc, int *status) {
  pdl_wait_then_release();
  const int l = threadIdx.x & 15;
  RowAt r;
  const bool live = row_at(n_kv, tokens, capacity, pos, counts, status, r);
  if (!__any_sync(0xffffffffu, live)) return;  // past a padded sequence's end
  float x[2][8] = {};
  if (live) {
    const size_t at = r.source_row * row_stride + (size_t)r.h * kD + 8 * l;
    load8(k + at, x[0]);
    load8(v + at, x[1]);
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    uint32_t dm;
    const uint32_t word = quantize8(x[kv], dm);
    if (!live) continue;
    uint32_t *o = reinterpret_cast<uint32_t *>((kv ? vc : kc) + r.cache_row * kRow);
    o[l] = word;
    if ((l & 3) == 0) o[16 + l / 4] = dm;
  }
}

// the lane's eight values of a cache row as fp16
__device__ __forceinline__ uint4 dequant8(const uint8_t *row, int l) {
  const uint32_t w = *reinterpret_cast<const uint32_t *>(row + 4 * l);
  const float2 dm = __half22float2(*reinterpret_cast<const __half2 *>(row + 64 + 4 * (l / 4)));
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = fmaf(dm.x, (float)((w >> (8 * i)) & 15u), dm.y);
    const float b = fmaf(dm.x, (float)((w >> (8 * i + 4)) & 15u), dm.y);
    const __half2 h = __floats2half2_rn(a, b);
    o[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

__global__ void __launch_bounds__(kThreads) kv4_read_kernel(
    const uint8_t *kc, const uint8_t *vc, int n_kv, int tokens, int capacity, const int32_t *pos,
    const int32_t *counts, __half *k, __half *v, int *status) {
  pdl_wait_then_release();
  const int l = threadIdx.x & 15;
  RowAt r;
  if (!row_at(n_kv, tokens, capacity, pos, counts, status, r)) return;
  const size_t at = (r.source_row * n_kv + r.h) * kD + 8 * l;
  const uint4 ok = dequant8(kc + r.cache_row * kRow, l);
  const uint4 ov = dequant8(vc + r.cache_row * kRow, l);
  *reinterpret_cast<uint4 *>(k + at) = ok;
  *reinterpret_cast<uint4 *>(v + at) = ov;
}

dim3 row_grid(const mlm_kv4_cache &c, int tokens) {
  return dim3((unsigned)(((long long)c.n_kv_heads * tokens + kRowsPerCta - 1) / kRowsPerCta),
              (unsigned)c.batch);
}

int check_rows(mlm_ctx *ctx, const mlm_kv4_cache *c, int tokens, const int32_t *pos,
               const int32_t *counts, const char *what) {
  const int st = kv4_check(ctx, c, what);
  if (st != MLM_OK) return st;
  MLM_REQUIRE(ctx, pos, MLM_ERR_ARG, "%s: null positions", what);
  MLM_REQUIRE(ctx, aligned4(pos) && aligned4(counts), MLM_ERR_ALIGN,
              "%s: positions and counts must be 4-byte aligned", what);
  MLM_REQUIRE(ctx, tokens > 0 && tokens <= c->capacity, MLM_ERR_SHAPE,
              "%s: tokens=%d (1 .. the capacity, %d)", what, tokens, c->capacity);
  MLM_REQUIRE(ctx, (long long)c->n_kv_heads * tokens <= 0x7FFFFFF0ll, MLM_ERR_SHAPE,
              "%s: %d KV heads x %d tokens in one call", what, c->n_kv_heads, tokens);
  return MLM_OK;
}

template <class T>
int append(mlm_ctx *ctx, const mlm_kv4_cache &c, const void *k, const void *v, int64_t row_stride,
           int tokens, const int32_t *pos, const int32_t *counts) {
  return check_launch_pdl(
      ctx,
      launch_pdl(kv4_append_kernel<T>, row_grid(c, tokens), dim3(kThreads), 0, ctx->stream,
                 reinterpret_cast<const T *>(k), reinterpret_cast<const T *>(v),
                 (long long)row_stride, c.n_kv_heads, tokens, c.capacity, pos, counts,
                 reinterpret_cast<uint8_t *>(c.k), reinterpret_cast<uint8_t *>(c.v),
                 ctx->dev_status),
      "mlm_kv4_append");
}

}  // namespace

int kv4_check(mlm_ctx *ctx, const mlm_kv4_cache *c, const char *what) {
  MLM_REQUIRE(ctx, c && c->k && c->v, MLM_ERR_ARG, "%s: null cache", what);
  MLM_REQUIRE(ctx, c->head_dim == kD, MLM_ERR_UNSUPPORTED,
              "%s: head_dim=%d (this build handles %d)", what, c->head_dim, kD);
  MLM_REQUIRE(ctx, c->batch > 0 && c->batch <= MLM_KV4_MAX_BATCH, MLM_ERR_SHAPE,
              "%s: batch=%d (1 .. %d)", what, c->batch, MLM_KV4_MAX_BATCH);
  MLM_REQUIRE(ctx, c->n_kv_heads > 0 && c->n_kv_heads <= 1024 && c->capacity > 0 &&
                       c->capacity <= (1 << 30),
              MLM_ERR_SHAPE, "%s: n_kv_heads=%d (1 .. 1024) capacity=%d (1 .. 2^30)", what,
              c->n_kv_heads, c->capacity);
  MLM_REQUIRE(ctx, (long long)c->batch * c->n_kv_heads * c->capacity <= (1ll << 32), MLM_ERR_SHAPE,
              "%s: batch=%d x n_kv_heads=%d x capacity=%d rows (at most 2^32)", what, c->batch,
              c->n_kv_heads, c->capacity);
  MLM_REQUIRE(ctx, aligned16(c->k) && aligned16(c->v), MLM_ERR_ALIGN,
              "%s: the cache must be 16-byte aligned", what);
  return MLM_OK;
}

}  // namespace mlm

using namespace mlm;

extern "C" int mlm_kv4_append(mlm_ctx *ctx, const mlm_kv4_cache *cache, const void *k,
                              const void *v, int type, int64_t row_stride, int tokens,
                              const int32_t *pos, const int32_t *counts) {
  MLM_CHECK_CTX(ctx);
  const int st = check_rows(ctx, cache, tokens, pos, counts, "mlm_kv4_append");
  if (st != MLM_OK) return st;
  MLM_REQUIRE(ctx, k && v, MLM_ERR_ARG, "mlm_kv4_append: null rows");
  MLM_REQUIRE(ctx, type == MLM_TYPE_F32 || type == MLM_TYPE_F16 || type == MLM_TYPE_BF16,
              MLM_ERR_UNSUPPORTED, "mlm_kv4_append: row type %d (F32 %d, F16 %d or BF16 %d)", type,
              MLM_TYPE_F32, MLM_TYPE_F16, MLM_TYPE_BF16);
  MLM_REQUIRE(ctx, row_stride >= (int64_t)cache->n_kv_heads * kD && row_stride <= (1ll << 31),
              MLM_ERR_SHAPE, "mlm_kv4_append: row_stride=%lld below %d heads x %d",
              (long long)row_stride, cache->n_kv_heads, kD);
  MLM_REQUIRE(ctx, aligned16(k) && aligned16(v) && row_stride % (type == MLM_TYPE_F32 ? 4 : 8) == 0,
              MLM_ERR_ALIGN, "mlm_kv4_append: rows must be 16-byte aligned");
  DeviceGuard guard(ctx);
  if (type == MLM_TYPE_F32) return append<float>(ctx, *cache, k, v, row_stride, tokens, pos, counts);
  if (type == MLM_TYPE_F16)
    return append<__half>(ctx, *cache, k, v, row_stride, tokens, pos, counts);
  return append<__nv_bfloat16>(ctx, *cache, k, v, row_stride, tokens, pos, counts);
}

extern "C" int mlm_kv4_read_f16(mlm_ctx *ctx, const mlm_kv4_cache *cache, int tokens,
                                const int32_t *pos, const int32_t *counts, void *k_out,
                                void *v_out) {
  MLM_CHECK_CTX(ctx);
  const int st = check_rows(ctx, cache, tokens, pos, counts, "mlm_kv4_read_f16");
  if (st != MLM_OK) return st;
  MLM_REQUIRE(ctx, k_out && v_out, MLM_ERR_ARG, "mlm_kv4_read_f16: null output");
  MLM_REQUIRE(ctx, aligned16(k_out) && aligned16(v_out), MLM_ERR_ALIGN,
              "mlm_kv4_read_f16: outputs must be 16-byte aligned");
  DeviceGuard guard(ctx);
  const mlm_kv4_cache &c = *cache;
  return check_launch_pdl(
      ctx,
      launch_pdl(kv4_read_kernel, row_grid(c, tokens), dim3(kThreads), 0, ctx->stream,
                 reinterpret_cast<const uint8_t *>(c.k), reinterpret_cast<const uint8_t *>(c.v),
                 c.n_kv_heads, tokens, c.capacity, pos, counts,
                 reinterpret_cast<__half *>(k_out), reinterpret_cast<__half *>(v_out),
                 ctx->dev_status),
      "mlm_kv4_read_f16");
}
