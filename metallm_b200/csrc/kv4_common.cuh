// kv4_common.cuh -- what the kernels on the 4-bit KV cache share: the sequences' shapes as
// read from device memory, the report of a bad one, small conversions.
#pragma once

#include "mlm_device.cuh"
#include "mlm_internal.h"

namespace mlm {

constexpr int kKv4Row = MLM_KV4_ROW_BYTES;
constexpr int kKv4D = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInvSqrtD = 0.08838834764831845f;  // 1 / sqrt(128)

// One mlm_attn_kv4 call.  Pointers to data that earlier kernels write carry no
// __restrict__, so that no load of it moves above the dependent wait.
struct Kv4AttnArgs {
  const uint8_t *kc, *vc;
  const __half *q;
  void *out;
  const int32_t *lens, *counts;
  float *parts;   // partial sums of heads that several CTAs share
  int *arrivals;  // [CTAs], zero between launches
  int *plan;      // many rows: the cut, for the kernel that joins the parts
  int *status;
  int batch, tokens, n_heads, n_kv, group, capacity;
};

// the sequence's rows and tokens, kept within the cache and the call
__device__ __forceinline__ void seq_shape(const Kv4AttnArgs &a, int b, int &len, int &count) {
  len = min(max(a.lens[b], 0), a.capacity);
  count = a.counts ? min(max(a.counts[b], 0), a.tokens) : a.tokens;
}
__device__ __forceinline__ bool seq_outside(const Kv4AttnArgs &a, int b) {
  return a.lens[b] < 0 || a.lens[b] > a.capacity ||
         (a.counts && (a.counts[b] < 0 || a.counts[b] > a.tokens));
}

// a position, length or count outside its cache, unless the word already tells of a worse
// failure (a wait that ran out)
__device__ __forceinline__ void report_outside(int *status) { atomicCAS(status, 0, MLM_ERR_SHAPE); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
__device__ __forceinline__ float low_f16(uint32_t v) {
  return __half2float(__ushort_as_half((unsigned short)v));
}
__device__ __forceinline__ uint32_t u4_get(const uint4 &v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// whether a (d, m) pair holds an infinity or NaN
__device__ __forceinline__ bool not_finite(uint32_t dm) {
  return (dm & 0x7C00u) == 0x7C00u || (dm & 0x7C000000u) == 0x7C000000u;
}

// kv4_attn.cu: up to 16 (token, head) rows per KV head; kv4_attn_many.cu: more
int kv4_attn_few(mlm_ctx *ctx, const Kv4AttnArgs &a, int out_type);
int kv4_attn_many(mlm_ctx *ctx, const Kv4AttnArgs &a, int out_type);
int kv4_attn_many_init(mlm_ctx *ctx);
size_t kv4_many_parts_bytes(int sm_count);
constexpr int kKv4PlanInts = 2 * (MLM_KV4_MAX_BATCH + 2);  // 64-bit: quota, the sequences' offsets

}  // namespace mlm
