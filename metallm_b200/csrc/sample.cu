// sample.cu -- one token per row of logits by temperature, top-k, top-p and
// min-p from a given random number: the sampling that stands beside the argmax
// of the reference's loop (ContentView.swift:124-146).
//
// With w_i = exp((x_i - max) / T) every filter keeps a prefix of the order
// "falling logit, then rising index", so a row needs one cut in that order, and
// a token is the 64-bit key (order-preserving bits of x, ~index): keep the keys
// >= the cut.  No sort of the row:
//  - masses are integers, w scaled to as many bits as the row's length leaves
//    free, so sums do not depend on their order and a row's token does not
//    depend on the run;
//  - a pass puts every kept token into one of 2048 bins of (max - x), sums
//    counts and masses per bin, and a scan finds the bin in which the k-th
//    token, or the top_p share of the mass, falls; that bin's tokens (tens, in
//    real logits) go into a list, are ranked, and give the exact cut.  A bin
//    with more tokens than the list holds (flat or constant rows) is first
//    narrowed by 11-bit digits of the key, which always ends, as keys are
//    distinct;
//  - the draw is by index: masses per warp's stretch of the row, a scan, and the
//    one stretch that holds the point is walked again.
// One cluster of CTAs per row; a CTA keeps its slice of the row in shared memory
// (read once) where it fits and reads it again from L2 where it does not.
#include <cooperative_groups.h>

#include <algorithm>

#include "mlm_device.cuh"
#include "mlm_internal.h"

namespace cg = cooperative_groups;

namespace mlm {
namespace {

using u64 = unsigned long long;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kCand = 1024;      // tokens of the list that is ranked
constexpr int kMaxCluster = 8;
constexpr u64 kAll = 1ull << 32;  // the smallest key of a logit that is not NaN

struct Shared {
  uint32_t cnt[kBins], lo[kBins], hi[kBins];  // this CTA's bins; masses as 64 bits in halves
  uint32_t g_cnt[kBins];                      // rank 0: the row's bins
  u64 g_mass[kBins];
  u64 cand[kCand], sorted[kCand];  // rank 0: tokens of the cut's bin
  u64 warp_mass[kWarps], warp_best[kWarps];
  uint32_t warp_cnt[kWarps];
  u64 best, mass;   // this CTA's largest key, kept mass
  int n_cand;       // rank 0
  // a pass's result, written to every CTA by rank 0
  int bin;
  uint32_t bin_cnt, above_cnt;
  u64 above_mass, target, cut;
};

__device__ __forceinline__ uint32_t order_bits(float v) {  // 0 for NaN
  if (v != v) return 0;
  const uint32_t b = __float_as_uint(__fadd_rn(v, 0.0f));  // -0 -> +0: equal values tie
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ u64 token_key(float v, int i) {
  return ((u64)order_bits(v) << 32) | (uint32_t)~(uint32_t)i;
}
// floor(f * m) for f in [0, 1)
__device__ __forceinline__ u64 fraction_of(float f, u64 m, bool up) {
  const u64 fix = (u64)((double)f * 18446744073709551616.0);  // exact down to 2^-40
  return __umul64hi(fix, m) + (up && fix * m != 0 ? 1 : 0);
}

struct Weights {
  float top;        // the row's largest logit
  double inv_t, scale;
  // w of a logit that is not NaN
  __device__ __forceinline__ double w(float x) const {
    if (top == INFINITY) return x == INFINITY ? 1.0 : 0.0;
    if (x == -INFINITY) return 0.0;
    return exp(((double)x - (double)top) * inv_t);
  }
  __device__ __forceinline__ u64 mass(double w) const { return __double2ull_rn(w * scale); }
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Row {
  cg::cluster_group cl;
  Shared &s;
  const float *x;  // the slice: shared memory, or the row in global memory
  int base, len;   // the slice's first token and length
  int w0, w1;      // this warp's stretch of the slice
  int rank, ctas;

  __device__ __forceinline__ void clear_bins() {
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.cnt[i] = s.lo[i] = s.hi[i] = 0;
    if (rank == 0 && threadIdx.x == 0) s.n_cand = 0;
    __syncthreads();
  }
  __device__ __forceinline__ void add(int bin, uint32_t n, u64 m) {
    if (n) atomicAdd(&s.cnt[bin], n);
    if (!m) return;
    const uint32_t lo = (uint32_t)m;
    uint32_t hi = (uint32_t)(m >> 32);
    if (atomicAdd(&s.lo[bin], lo) + lo < lo) ++hi;  // carry
    if (hi) atomicAdd(&s.hi[bin], hi);
  }

  // Sum the CTAs' bins and find the first at which the running count reaches
  // `k` (k > 0), or the running mass (k == 0) the target; the target is s.target or,
  // when top_p is not NaN, the top_p share of the sum of all bins.  `first`:
  // what lies above the bins.  The result lands in every CTA's s.bin (-1: never
  // reached), s.bin_cnt, s.above_*.
  __device__ void find(uint32_t k, float top_p, uint32_t first_cnt, u64 first_mass) {
    cl.sync();  // every CTA's bins are complete
    const int per = kBins / ctas;
    for (int i = threadIdx.x; i < per; i += kThreads) {
      const int bin = rank * per + i;
      uint32_t c = 0;
      u64 m = 0;
      for (int r = 0; r < ctas; ++r) {
        c += *cl.map_shared_rank(&s.cnt[bin], r);
        m += (u64)*cl.map_shared_rank(&s.lo[bin], r) +
             ((u64)*cl.map_shared_rank(&s.hi[bin], r) << 32);
      }
      *cl.map_shared_rank(&s.g_cnt[bin], 0) = c;
      *cl.map_shared_rank(&s.g_mass[bin], 0) = m;
    }
    cl.sync();
    if (rank == 0) {
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
      constexpr int kPer = kBins / kThreads;
      uint32_t c[kPer], csum = 0;
      u64 m[kPer], msum = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        c[i] = s.g_cnt[threadIdx.x * kPer + i];
        m[i] = s.g_mass[threadIdx.x * kPer + i];
        csum += c[i];
        msum += m[i];
      }
      uint32_t cin = csum;
      u64 min_ = msum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t cu = __shfl_up_sync(0xffffffffu, cin, o);
        const u64 mu = __shfl_up_sync(0xffffffffu, min_, o);
        if (lane >= o) {
          cin += cu;
          min_ += mu;
        }
      }
      if (lane == 31) {
        s.warp_cnt[warp] = cin;
        s.warp_mass[warp] = min_;
      }
      if (threadIdx.x == 0) s.bin = -1;
      __syncthreads();
      uint32_t cb = first_cnt;
      u64 mb = first_mass, total = first_mass;
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) {
          cb += s.warp_cnt[w];
          mb += s.warp_mass[w];
        }
        total += s.warp_mass[w];
      }
      u64 target = s.target;
      if (top_p == top_p) target = max(fraction_of(fmaxf(top_p, 0.f), total, true), 1ull);
      cb += cin - csum;
      mb += min_ - msum;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const bool here = k ? (cb < k && cb + c[i] >= k) : (mb < target && mb + m[i] >= target);
        if (here) {
          s.bin = threadIdx.x * kPer + i;
          s.bin_cnt = c[i];
          s.above_cnt = cb;
          s.above_mass = mb;
          s.target = target;
        }
        cb += c[i];
        mb += m[i];
      }
      __syncthreads();
      if (threadIdx.x > 0 && threadIdx.x < ctas) {
        Shared *o = cl.map_shared_rank(&s, threadIdx.x);
        o->bin = s.bin;
        o->bin_cnt = s.bin_cnt;
        o->above_cnt = s.above_cnt;
        o->above_mass = s.above_mass;
        o->target = s.target;
      }
    }
    cl.sync();
  }

  // The cut of the first k tokens (k > 0) or of the shortest prefix that holds
  // the top_p share of the mass, among the keys >= `within`: every CTA
  // returns the key of the last kept token.
  __device__ u64 cut(uint32_t k, float top_p, u64 within, const Weights &W, float bin_scale) {
    auto value_bin = [&](float v) {
      if (v == W.top) return 0;
      return (int)fminf((W.top - v) * bin_scale, (float)(kBins - 1));
    };
    clear_bins();
    {
      // the last bin also takes all that lies below the range: summed in
      // registers first, as half the row may fall there
      uint32_t rest_n = 0;
      u64 rest_m = 0;
#pragma unroll 4
      for (int i = threadIdx.x; i < len; i += kThreads) {
        const float v = x[i];
        const u64 key = token_key(v, base + i);
        if (key < within) continue;
        const u64 m = k ? 0 : W.mass(W.w(v));
        const int bin = value_bin(v);
        if (bin < kBins - 1) {
          add(bin, 1, m);
        } else {
          ++rest_n;
          rest_m += m;
        }
      }
      rest_n = __reduce_add_sync(0xffffffffu, rest_n);
      rest_m = warp_sum64(rest_m);
      if ((threadIdx.x & 31) == 0) add(kBins - 1, rest_n, rest_m);
    }
    find(k, top_p, 0, 0);
    if (s.bin < 0) return within;  // fewer than k tokens: all of them
    const int vbin = s.bin;
    // narrow a crowded bin by digits of the key, highest first
    int shift = 64, bits = 0;
    u64 prefix = 0;
    auto inside = [&](float v, u64 key) {
      return key >= within && value_bin(v) == vbin && (shift == 64 || (key >> shift) == prefix);
    };
    while (s.bin_cnt > kCand) {
      bits = min(11, shift);
      const uint32_t above_cnt = s.above_cnt;
      const u64 above_mass = s.above_mass;
      clear_bins();
      for (int i = threadIdx.x; i < len; i += kThreads) {
        const float v = x[i];
        const u64 key = token_key(v, base + i);
        if (!inside(v, key)) continue;
        const int digit = (int)((key >> (shift - bits)) & ((1u << bits) - 1));
        add((1 << bits) - 1 - digit, 1, k ? 0 : W.mass(W.w(v)));
      }
      find(k, NAN, above_cnt, above_mass);
      prefix = (prefix << bits) | (u64)((1 << bits) - 1 - s.bin);
      shift -= bits;
    }
    // the bin's tokens into rank 0's list, in any order
    int *n_cand = cl.map_shared_rank(&s.n_cand, 0);
    u64 *cand = cl.map_shared_rank(&s.cand[0], 0);
    for (int i = threadIdx.x; i < len; i += kThreads) {
      const float v = x[i];
      const u64 key = token_key(v, base + i);
      if (inside(v, key)) cand[atomicAdd(n_cand, 1)] = key;
    }
    cl.sync();
    if (rank == 0) {
      const int n = s.n_cand;
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const u64 key = s.cand[i];
        int place = 0;
        for (int j = 0; j < n; ++j) place += s.cand[j] > key;
        s.sorted[place] = key;
      }
      __syncthreads();
      if (k) {
        if (threadIdx.x == 0) s.cut = s.sorted[k - s.above_cnt - 1];
      } else if (threadIdx.x < 32) {
        // one warp walks the ranked tokens until the mass is reached
        u64 run = s.above_mass;
        u64 found = s.sorted[n - 1];
        for (int i0 = 0; i0 < n; i0 += 32) {
          const int i = i0 + threadIdx.x;
          u64 m = i < n ? W.mass(W.w(order_value((uint32_t)(s.sorted[i] >> 32)))) : 0;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const u64 up = __shfl_up_sync(0xffffffffu, m, o);
            if ((int)threadIdx.x >= o) m += up;
          }
          const uint32_t hit = __ballot_sync(0xffffffffu, i < n && run + m >= s.target);
          if (hit) {
            found = s.sorted[i0 + __ffs(hit) - 1];
            break;
          }
          run += __shfl_sync(0xffffffffu, m, 31);
        }
        if (threadIdx.x == 0) s.cut = found;
      }
      __syncthreads();
      if (threadIdx.x > 0 && threadIdx.x < ctas) cl.map_shared_rank(&s, threadIdx.x)->cut = s.cut;
    }
    cl.sync();
    return s.cut;
  }
};

__global__ void __launch_bounds__(kThreads) sample_kernel(
    const float *logits, int n, long long row_stride, int slice, int resident, int mass_bits,
    const mlm_sample_params *params, const float *uniform, int32_t *token, float *prob) {
  extern __shared__ __align__(16) uint8_t s_raw[];
  Shared &s = *reinterpret_cast<Shared *>(s_raw);
  float *s_x = reinterpret_cast<float *>(s_raw + sizeof(Shared));
  pdl_wait_then_release();
  cg::cluster_group cl = cg::this_cluster();
  const int rank = cl.block_rank(), ctas = cl.num_blocks();
  const int row = blockIdx.x / ctas;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int base = min(n, rank * slice), len = min(n - base, slice);
  const float *g = logits + row * row_stride + base;
  const int per = (len + kWarps * 32 - 1) / (kWarps * 32) * 32;
  Row r{cl, s, resident ? s_x : g, base, len, min(len, warp * per), min(len, (warp + 1) * per),
        rank, ctas};

  // the slice into shared memory; the row's largest key
  u64 best = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < len; i += kThreads) {
    const float v = g[i];
    if (resident) s_x[i] = v;
    const u64 key = token_key(v, base + i);
    best = key > best ? key : best;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) s.warp_best[warp] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWarps; ++w) best = max(best, s.warp_best[w]);
    s.best = best;
  }
  cl.sync();
  best = 0;
  for (int q = 0; q < ctas; ++q) best = max(best, *cl.map_shared_rank(&s.best, q));

  const mlm_sample_params p = params[row];
  const float top = order_value((uint32_t)(best >> 32));
  const bool none = best < kAll || top == -INFINITY;
  if (none || !(p.temperature > 0.f)) {
    if (rank == 0 && threadIdx.x == 0) {
      // only NaN: 0, as the argmax
      token[row] = best < kAll ? 0 : (int32_t)~(uint32_t)best;
      if (prob) prob[row] = none ? 0.f : 1.f;
    }
    cl.sync();  // no CTA leaves while another may still read its s.best
    return;
  }
  Weights W;
  W.top = top;
  W.inv_t = 1.0 / (double)p.temperature;
  W.scale = (double)(1ull << mass_bits);
  u64 cut = kAll;
  // bins over the logits that matter: 24 temperatures, but at least 16 and at
  // most 64 below the largest
  const float bin_scale = (float)kBins / fminf(fmaxf(24.f * p.temperature, 16.f), 64.f);
  if (p.top_k > 0 && p.top_k < n) cut = r.cut((uint32_t)p.top_k, NAN, cut, W, bin_scale);
  if (p.top_p < 1.f) cut = r.cut(0, p.top_p, cut, W, bin_scale);

  // the kept mass of every warp's stretch
  const double min_w = p.min_p > 0.f ? fmin((double)p.min_p, 1.0) : 0.0;
  auto kept = [&](int i) -> u64 {
    const float v = r.x[i];
    if (token_key(v, base + i) < cut) return 0;
    const double w = W.w(v);
    return w >= min_w ? W.mass(w) : 0;
  };
  u64 m = 0;
#pragma unroll 4
  for (int i = r.w0 + lane; i < r.w1; i += 32) m += kept(i);
  m = warp_sum64(m);
  if (lane == 0) s.warp_mass[warp] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    u64 t = 0;
    for (int w = 0; w < kWarps; ++w) t += s.warp_mass[w];
    s.mass = t;
  }
  cl.sync();
  u64 before = 0, total = 0;
  for (int q = 0; q < ctas; ++q) {
    const u64 t = *cl.map_shared_rank(&s.mass, q);
    if (q < rank) before += t;
    total += t;
  }
  float u = uniform[row];
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;  // NaN: 0
  const u64 point = fraction_of(u, total, false);  // the first token whose running mass exceeds it
  for (int w = 0; w < warp; ++w) before += s.warp_mass[w];
  if (point >= before && point < before + m) {
    u64 run = before;
    for (int i0 = r.w0; i0 < r.w1; i0 += 32) {
      const int i = i0 + lane;
      u64 t = i < r.w1 ? kept(i) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 up = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += up;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, run + t > point);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          token[row] = base + i;
          if (prob) prob[row] = (float)(W.w(r.x[i]) * W.scale / (double)total);
        }
        break;
      }
      run += __shfl_sync(0xffffffffu, t, 31);
    }
  }
  cl.sync();  // no CTA leaves while another may still read its s.mass
}

constexpr int kMaxN = 1 << 22;
// shared memory a slice may take beside the bins (one CTA per SM)
constexpr size_t kSliceBytes = 160 * 1024;

}  // namespace

int sample_init(mlm_ctx *ctx) {
  MLM_CUDA_TRY(ctx, cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)(sizeof(Shared) + kSliceBytes)));
  return MLM_OK;
}

}  // namespace mlm

using namespace mlm;

extern "C" int mlm_sample_f32(mlm_ctx *ctx, const float *logits, int rows, int n,
                              int64_t row_stride, const mlm_sample_params *params,
                              const float *uniform, int32_t *token, float *prob) {
  MLM_CHECK_CTX(ctx);
  MLM_REQUIRE(ctx, logits && params && uniform && token, MLM_ERR_ARG, "mlm_sample_f32: null buffer");
  MLM_REQUIRE(ctx, rows > 0 && rows <= 65536 && n > 0 && n <= kMaxN, MLM_ERR_SHAPE,
              "mlm_sample_f32: rows=%d (1 .. 65536) n=%d (1 .. %d)", rows, n, kMaxN);
  MLM_REQUIRE(ctx, row_stride >= n || rows == 1, MLM_ERR_SHAPE,
              "mlm_sample_f32: row_stride=%lld below n=%d", (long long)row_stride, n);
  MLM_REQUIRE(ctx, aligned4(logits) && aligned4(params) && aligned4(uniform) && aligned4(token) &&
                       aligned4(prob),
              MLM_ERR_ALIGN, "mlm_sample_f32: buffers must be 4-byte aligned");
  DeviceGuard guard(ctx);
  int ctas = kMaxCluster;
  while (ctas > 1 && (rows * ctas > ctx->sm_count || n < 2048 * ctas)) ctas /= 2;
  const int slice = (n + ctas - 1) / ctas;
  const int resident = (size_t)slice * 4 <= kSliceBytes;
  int bits = 62;
  while ((1ll << (62 - bits)) < n) --bits;
  bits = std::min(bits, 50);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared) + (resident ? (size_t)slice * 4 : 0);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return check_launch_pdl(ctx,
                          cudaLaunchKernelEx(&cfg, sample_kernel, logits, n, (long long)row_stride,
                                             slice, resident, bits, params, uniform, token, prob),
                          "mlm_sample_f32");
}
