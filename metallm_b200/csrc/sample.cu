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
//  - a pass puts every token into one of 2048 bins of (max - x), sums counts or
//    masses per bin, and a scan finds the bin in which the k-th token, or the
//    top_p share of the mass, falls.  Where the tokens down to that bin fit a list
//    (tens, for usual settings) they are gathered and one CTA does the rest on the
//    list: ranks by counting, masses, both cuts and the draw.  Otherwise the bin's
//    tokens alone are gathered and give the exact cut, and the draw goes over the
//    row again; a bin with more tokens than the list holds (flat or constant rows)
//    is first narrowed by 11-bit digits of the key, which always ends, as keys are
//    distinct;
//  - the draw is by index: masses per warp's stretch of the row, a scan, and the
//    one stretch that holds the point is walked again by the whole CTA.
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

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kCand = 1024;       // tokens of the list
constexpr int kMaxCluster = 16;   // of CTAs; above 8 needs the opt-in
constexpr int kMinSlice = 4096;   // tokens per CTA that are worth a CTA
constexpr u64 kAll = 1ull << 32;  // the smallest key of a logit that is not NaN

struct Shared {
  double exp2_64[64];                         // 2^(j/64)
  uint32_t cnt[kBins], lo[kBins], hi[kBins];  // this CTA's bins; masses as 64 bits in halves
  uint32_t g_cnt[kBins];                      // rank 0: the row's bins
  u64 g_mass[kBins];
  // rank 0: the list, in order of arrival, then ranked (by key, later by index)
  __align__(16) u64 cand[kCand];
  u64 sorted[kCand];
  __align__(16) uint32_t place[kCand];
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
// floor(f * m) for f in [0, 1), or its ceiling
__device__ __forceinline__ u64 fraction_of(float f, u64 m, bool up) {
  const u64 fix = (u64)((double)f * 18446744073709551616.0);  // exact down to 2^-40
  return __umul64hi(fix, m) + (up && fix * m != 0 ? 1 : 0);
}

struct Weights {
  float top;           // the row's largest logit
  double octaves;      // 64 log2(e) / T: (x - top) in 64ths of an octave
  double scale;        // mass of w = 1
  int mass_bits;       // its power of two
  const double *table;

  // w of a logit that is not NaN, to 2^-44: with y = 64 log2 w split into an
  // integer k and |f| <= 1/2, w = 2^(k >> 6) 2^((k & 63) / 64) e^r for r = f ln2 / 64,
  // e^r by its series to r^4 (r^5 / 120 < 2^-44).  (Table look-up and a short
  // series: P. T. P. Tang, ACM TOMS 15(2), 1989.)
  __device__ __forceinline__ double w(float x) const { return w_scaled(x, 0); }
  // w 2^bits
  __device__ __forceinline__ double w_scaled(float x, int bits) const {
    if (top == INFINITY) return x == INFINITY ? (bits ? scale : 1.0) : 0.0;
    if (x == -INFINITY) return 0.0;
    constexpr double kMagic = 6755399441055744.0;  // 1.5 2^52: the sum's low word is round(y)
    constexpr double kC = 0.010830424696249145;    // ln2 / 64
    const double y = fmax(((double)x - (double)top) * octaves, -60000.0);
    const double kd = y + kMagic;
    const int k = __double2loint(kd);
    const double f = y - (kd - kMagic);
    double e = fma(f, kC * kC * kC * kC / 24, kC * kC * kC / 6);
    e = fma(f, e, kC * kC / 2);
    e = fma(f, e, kC);
    e *= f;
    const double t = table[k & 63];
    const double v = fma(t, e, t);
    return __hiloint2double(__double2hiint(v) + (((k >> 6) + bits) << 20), __double2loint(v));
  }
  // round(w 2^mass_bits), below 2^51
  __device__ __forceinline__ u64 mass(float x) const {
    const double v = w_scaled(x, mass_bits) + 4503599627370496.0;  // 2^52
    return (u64)__double_as_longlong(v) & 0xFFFFFFFFFFFFFull;
  }
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// inclusive sums over the lanes
__device__ __forceinline__ u64 warp_scan64(u64 v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}
// the exclusive sum of the lanes' (= warps') values before this warp's, and their total
__device__ __forceinline__ u64 before_warp(const u64 *v, u64 &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const u64 in = warp_scan64(v[lane]);
  total = __shfl_sync(0xffffffffu, in, 31);
  return __shfl_sync(0xffffffffu, in, warp) - v[warp];
}
static_assert(kWarps == 32, "a lane per warp");

struct Row {
  cg::cluster_group cl;
  Shared &s;
  const float *x;  // the slice: shared memory, or the row in global memory
  int base, len;   // the slice's first token and length
  int rank, ctas;

  template <class F>
  __device__ __forceinline__ void each(F f) {
    int i = threadIdx.x;
    for (; i + 3 * kThreads < len; i += 4 * kThreads) {
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = x[i + k * kThreads];
#pragma unroll
      for (int k = 0; k < 4; ++k) f(v[k], i + k * kThreads);
    }
    for (; i < len; i += kThreads) f(x[i], i);
  }
  __device__ __forceinline__ void clear_bins(bool masses) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      s.cnt[i] = 0;
      s.lo[i] = 0;
      if (masses) s.hi[i] = 0;
    }
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
    if (ctas > 1)
      cl.sync();  // every CTA's bins are complete
    else
      __syncthreads();
    const int per = kBins / ctas;
    for (int i = threadIdx.x; i < per; i += kThreads) {
      const int bin = rank * per + i;
      uint32_t c = 0;
      u64 m = 0;
#pragma unroll 4
      for (int r = 0; r < ctas; ++r) {
        c += *cl.map_shared_rank(&s.cnt[bin], r);
        if (!k)
          m += (u64)*cl.map_shared_rank(&s.lo[bin], r) +
               ((u64)*cl.map_shared_rank(&s.hi[bin], r) << 32);
      }
      *cl.map_shared_rank(&s.g_cnt[bin], 0) = c;
      *cl.map_shared_rank(&s.g_mass[bin], 0) = m;
    }
    if (ctas > 1)
      cl.sync();
    else
      __syncthreads();
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
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t cu = __shfl_up_sync(0xffffffffu, cin, o);
        if (lane >= o) cin += cu;
      }
      const u64 min_ = warp_scan64(msum);
      if (lane == 31) {
        s.warp_cnt[warp] = cin;
        s.warp_mass[warp] = min_;
      }
      if (threadIdx.x == 0) s.bin = -1;
      __syncthreads();
      u64 total;
      u64 mb = first_mass + before_warp(s.warp_mass, total) + min_ - msum;
      total += first_mass;
      uint32_t cw = s.warp_cnt[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t cu = __shfl_up_sync(0xffffffffu, cw, o);
        if (lane >= o) cw += cu;
      }
      uint32_t cb = first_cnt + __shfl_sync(0xffffffffu, cw, warp) - s.warp_cnt[warp] + cin - csum;
      u64 target = s.target;
      if (top_p == top_p) target = max(fraction_of(fmaxf(top_p, 0.f), total, true), 1ull);
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
    if (ctas > 1)
      cl.sync();
    else
      __syncthreads();
  }

  // tokens of `pred` into rank 0's list, in any order
  template <class P>
  __device__ __forceinline__ void gather(P pred) {
    int *n_cand = cl.map_shared_rank(&s.n_cand, 0);
    u64 *cand = cl.map_shared_rank(&s.cand[0], 0);
    each([&](float v, int i) {
      const u64 key = token_key(v, base + i);
      if (pred(v, key)) cand[atomicAdd(n_cand, 1)] = key;
    });
    if (ctas > 1)
      cl.sync();
    else
      __syncthreads();
  }

  // rank 0: the list in order of falling keys into s.sorted.  A token's place is
  // the number of larger keys, counted by as many threads as the block has to spare.
  __device__ void rank_list(int n) {
    int share = 1;
    while (2 * share * n <= kThreads) share *= 2;
    for (int i = threadIdx.x; i < n; i += kThreads) s.place[i] = 0;
    __syncthreads();
    for (int t = threadIdx.x; t < n * share; t += kThreads) {
      const int i = t / share, j0 = t - i * share;
      const u64 key = s.cand[i];
      uint32_t c = 0;
#pragma unroll 4
      for (int j = j0; j < n; j += share) c += s.cand[j] > key;
      if (c) atomicAdd(&s.place[i], c);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) s.sorted[s.place[i]] = s.cand[i];
    __syncthreads();
  }

  // The cut of the first k tokens (k > 0) or of the shortest prefix that holds
  // the top_p share of the mass, among the keys >= `within`: every CTA
  // returns the key of the last kept token.  Where `listed` is given and the tokens
  // down to the cut's bin fit the list, they are left there instead (*listed set).
  __device__ u64 cut(uint32_t k, float top_p, u64 within, const Weights &W, float bin_scale,
                     bool *listed) {
    auto value_bin = [&](float v) {
      if (v == W.top) return 0;
      return (int)fminf((W.top - v) * bin_scale, (float)(kBins - 1));
    };
    clear_bins(!k);
    {
      // the last bin also takes all that lies below the range: summed in
      // registers first, as half the row may fall there
      uint32_t rest_n = 0;
      u64 rest_m = 0;
      each([&](float v, int i) {
        const u64 key = token_key(v, base + i);
        if (key < within) return;
        const u64 m = k ? 0 : W.mass(v);
        const int bin = value_bin(v);
        if (bin < kBins - 1) {
          add(bin, 1, m);
        } else {
          ++rest_n;
          rest_m += m;
        }
      });
      rest_n = __reduce_add_sync(0xffffffffu, rest_n);
      rest_m = warp_sum64(rest_m);
      if ((threadIdx.x & 31) == 0) add(kBins - 1, rest_n, rest_m);
    }
    find(k, top_p, 0, 0);
    if (s.bin < 0) return within;  // fewer than k tokens: all of them
    const int vbin = s.bin;
    if (listed && s.above_cnt + s.bin_cnt <= kCand) {
      *listed = true;
      gather([&](float v, u64 key) { return key >= within && value_bin(v) <= vbin; });
      return within;
    }
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
      clear_bins(!k);
      each([&](float v, int i) {
        const u64 key = token_key(v, base + i);
        if (!inside(v, key)) return;
        const int digit = (int)((key >> (shift - bits)) & ((1u << bits) - 1));
        add((1 << bits) - 1 - digit, 1, k ? 0 : W.mass(v));
      });
      find(k, NAN, above_cnt, above_mass);
      prefix = (prefix << bits) | (u64)((1 << bits) - 1 - s.bin);
      shift -= bits;
    }
    gather(inside);
    if (rank == 0) {
      const int n = s.n_cand;
      rank_list(n);
      if (k) {
        if (threadIdx.x == 0) s.cut = s.sorted[k - s.above_cnt - 1];
      } else if (threadIdx.x < 32) {
        // one warp walks the ranked tokens until the mass is reached
        u64 run = s.above_mass;
        u64 found = s.sorted[n - 1];
        for (int i0 = 0; i0 < n; i0 += 32) {
          const int i = i0 + threadIdx.x;
          const u64 m =
              warp_scan64(i < n ? W.mass(order_value((uint32_t)(s.sorted[i] >> 32))) : 0);
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
    if (ctas > 1)
      cl.sync();
    else
      __syncthreads();
    return s.cut;
  }

  // rank 0: both cuts and the draw on the list.  top_p_target: the mass the top-p
  // prefix has to reach, or 0 to take the share of the first k tokens' mass.
  __device__ void draw_listed(uint32_t k, float top_p, u64 top_p_target, double min_w, float u,
                              const Weights &W, int32_t *token, float *prob) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = threadIdx.x;
    const int n = s.n_cand;
    rank_list(n);
    const int n_k = k ? min(n, (int)k) : n;
    const u64 key = i < n_k ? s.sorted[i] : 0;
    const float v = order_value((uint32_t)(key >> 32));
    const u64 m = i < n_k ? W.mass(v) : 0;
    u64 in = warp_scan64(m), total;
    if (lane == 31) s.warp_mass[warp] = in;
    __syncthreads();
    in += before_warp(s.warp_mass, total);
    if (!top_p_target && top_p < 1.f)
      top_p_target = max(fraction_of(fmaxf(top_p, 0.f), total, true), 1ull);
    // the kept ones are the first of the ranked ones
    const bool keep = i < n_k && (!top_p_target || in - m < top_p_target) && W.w(v) >= min_w;
    const int n_keep = __syncthreads_count(keep);
    if (keep) {  // ranked again, by index: the low word of a key is ~index
      s.cand[i] = (key << 32) | (uint32_t)i;
      s.g_mass[i] = m;
    }
    __syncthreads();
    rank_list(n_keep);
    const uint32_t at = i < n_keep ? (uint32_t)s.sorted[i] & (kCand - 1) : 0;
    const u64 mine = i < n_keep ? s.g_mass[at] : 0;
    in = warp_scan64(mine);
    if (lane == 31) s.warp_mass[warp] = in;
    __syncthreads();
    in += before_warp(s.warp_mass, total);
    const u64 point = fraction_of(u, total, false);
    if (in > point && in - mine <= point) {  // one thread: its mass is not 0
      const uint32_t index = ~(uint32_t)(s.sorted[i] >> 32);
      *token = (int32_t)index;
      if (prob) s.target = at;
    }
    if (prob) {  // w itself over the kept mass
      __syncthreads();
      if (i == (int)s.target) *prob = (float)(W.w_scaled(v, W.mass_bits) / (double)total);
    }
  }
};

__global__ void __launch_bounds__(kThreads, 1) sample_kernel(
    const float *logits, int n, long long row_stride, int slice, int resident, int mass_bits,
    const mlm_sample_params *params, const float *uniform, int32_t *token, float *prob) {
  extern __shared__ __align__(16) uint8_t s_raw[];
  Shared &s = *reinterpret_cast<Shared *>(s_raw);
  float *s_x = reinterpret_cast<float *>(s_raw + sizeof(Shared));
  if (threadIdx.x < 64) s.exp2_64[threadIdx.x] = exp2(threadIdx.x / 64.0);
  pdl_wait_then_release();
  cg::cluster_group cl = cg::this_cluster();
  const int rank = cl.block_rank(), ctas = cl.num_blocks();
  const int row = blockIdx.x / ctas;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int base = min(n, rank * slice), len = min(n - base, slice);
  const float *g = logits + row * row_stride + base;
  const mlm_sample_params p = params[row];
  Row r{cl, s, g, base, len, rank, ctas};

  // the slice into shared memory; the row's largest key
  u64 best = 0;
  r.each([&](float v, int i) {
    if (resident) s_x[i] = v;
    const u64 key = token_key(v, base + i);
    best = key > best ? key : best;
  });
  if (resident) r.x = s_x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) s.warp_best[warp] = best;
  __syncthreads();
  best = s.warp_best[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (ctas > 1) {
    if (threadIdx.x == 0) s.best = best;
    cl.sync();
    best = *cl.map_shared_rank(&s.best, lane < ctas ? lane : 0);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  }

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
  W.octaves = 92.332482616893656 / (double)p.temperature;  // 64 log2(e) / T
  W.scale = (double)(1ull << mass_bits);
  W.mass_bits = mass_bits;
  W.table = s.exp2_64;
  // bins over the logits that matter: 24 temperatures, but at least 16 and at
  // most 64 below the largest
  const float bin_scale = (float)kBins / fminf(fmaxf(24.f * p.temperature, 16.f), 64.f);
  const uint32_t k = p.top_k > 0 && p.top_k < n ? (uint32_t)p.top_k : 0;
  const double min_w = p.min_p > 0.f ? fmin((double)p.min_p, 1.0) : 0.0;
  float u = uniform[row];
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;  // NaN: 0
  u64 cut = kAll;
  bool listed = false;
  if (k) cut = r.cut(k, NAN, cut, W, bin_scale, &listed);
  if (p.top_p < 1.f && !listed) cut = r.cut(0, p.top_p, cut, W, bin_scale, k ? nullptr : &listed);
  if (listed) {
    if (rank == 0)
      r.draw_listed(k, p.top_p, k ? 0 : s.target, min_w, u, W, token + row, prob ? prob + row : nullptr);
    return;  // the other CTAs' shared memory is no longer read (gather ended in a barrier)
  }

  // the kept mass of every warp's stretch
  auto kept = [&](float v, int i) -> u64 {
    if (token_key(v, base + i) < cut) return 0;
    return min_w == 0.0 || W.w(v) >= min_w ? W.mass(v) : 0;
  };
  // this warp's share of a range, 4 loads in flight
  auto range_mass = [&](int i0, int i1) -> u64 {
    u64 m = 0;
    int i = i0 + lane;
    for (; i + 96 < i1; i += 128) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = r.x[i + 32 * j];
#pragma unroll
      for (int j = 0; j < 4; ++j) m += kept(v[j], i + 32 * j);
    }
    for (; i < i1; i += 32) m += kept(r.x[i], i);
    return warp_sum64(m);
  };
  const int per = (len + kWarps * 32 - 1) / (kWarps * 32) * 32;
  u64 m = range_mass(min(len, warp * per), min(len, (warp + 1) * per));
  if (lane == 0) s.warp_mass[warp] = m;
  __syncthreads();
  u64 total;
  u64 before = before_warp(s.warp_mass, total);
  if (ctas > 1) {
    if (threadIdx.x == 0) s.mass = total;
    cl.sync();
    const u64 of = lane < ctas ? *cl.map_shared_rank(&s.mass, lane) : 0;
    const u64 in = warp_scan64(of);
    total = __shfl_sync(0xffffffffu, in, 31);
    before += __shfl_sync(0xffffffffu, in - of, rank);
  }
  const u64 point = fraction_of(u, total, false);  // the first token whose running mass exceeds it
  // the stretch that holds the point, 1/32 of it per warp, then 32 tokens at a time
  if (threadIdx.x == 0) s.bin = -1;
  __syncthreads();
  if (lane == 0 && point >= before && point < before + m) {
    s.bin = warp;
    s.target = before;
  }
  __syncthreads();
  if (s.bin >= 0) {
    const int a0 = min(len, s.bin * per), a1 = min(len, a0 + per);
    const int sub = (per + kWarps * 32 - 1) / (kWarps * 32) * 32;
    const int b0 = min(a1, a0 + warp * sub), b1 = min(a1, b0 + sub);
    before = s.target;
    m = range_mass(b0, b1);
    if (lane == 0) s.warp_mass[warp] = m;
    __syncthreads();
    u64 unused;
    before += before_warp(s.warp_mass, unused);
    if (point >= before && point < before + m) {
      for (int i0 = b0; i0 < b1; i0 += 32) {
        const int i = i0 + lane;
        const u64 t = warp_scan64(i < b1 ? kept(r.x[i], i) : 0);
        const uint32_t hit = __ballot_sync(0xffffffffu, before + t > point);
        if (hit) {
          if (lane == __ffs(hit) - 1) {
            token[row] = base + i;
            if (prob) prob[row] = (float)(W.w_scaled(r.x[i], mass_bits) / (double)total);
          }
          break;
        }
        before += __shfl_sync(0xffffffffu, t, 31);
      }
    }
  }
  if (ctas > 1) cl.sync();  // no CTA leaves while another may still read its s.mass
}

constexpr int kMaxN = 1 << 22;
// shared memory a slice may take beside the bins (one CTA per SM)
constexpr size_t kSliceBytes = 150 * 1024;
static_assert(sizeof(Shared) + kSliceBytes <= 227 * 1024, "a CTA's shared memory");

}  // namespace

int sample_init(mlm_ctx *ctx) {
  MLM_CUDA_TRY(ctx, cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)(sizeof(Shared) + kSliceBytes)));
  MLM_CUDA_TRY(ctx, cudaFuncSetAttribute(sample_kernel,
                                         cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
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
  while (ctas > 1 && (rows * ctas > ctx->sm_count || n < kMinSlice * ctas)) ctas /= 2;
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
