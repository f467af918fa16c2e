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
//    top_p share of the mass, falls.  For a short top-k each CTA does so for its own
//    slice and sends the slice's first k tokens to the row's first CTA, which sorts
//    them, takes masses, applies the cuts and draws: one exchange between the CTAs.
//    Otherwise the CTAs' bins are summed; where the tokens down to the cut's bin fit
//    the list the same CTA finishes on it, and where they do not the bin's tokens
//    alone are gathered and give the exact cut, and the draw goes over the row
//    again.  A bin with more tokens than the list holds (flat or constant rows) is
//    first narrowed by 11-bit digits of the key, which always ends, as keys are
//    distinct;
//  - the draw is by index: masses per warp's stretch of the row, a scan, and the
//    one stretch that holds the point is walked again by the whole CTA.
// Bound by the latency of these steps: one row of 128256 tokens with a top-k of 40 12.4
// us, 64 rows of mixed settings 56 to 71 us (by their values), with top-p alone 101 us;
// their bytes would take 0.1 and 5 us.  With 64 rows issue slots are 51 to 54 % busy, the
// ALU pipe a third, the fp64 pipe 11 %; the 256 CTAs, one per SM, take 1.7 waves.
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
constexpr int kMaxCluster = 8;
constexpr int kAhead = 8;         // logits of a thread in flight
constexpr int kMinSlice = 4096;   // tokens per CTA that are worth a CTA
constexpr u64 kAll = 1ull << 32;  // the smallest key of a logit that is not NaN

struct Shared {
  double exp2_256[256];                       // 2^(j/256)
  uint32_t cnt[kBins], lo[kBins], hi[kBins];  // this CTA's bins; masses as 64 bits in halves
  uint32_t g_cnt[kBins];                      // rank 0: the row's bins
  u64 g_mass[kBins];
  // rank 0: the list, in order of arrival, then ranked (by key, later by index)
  u64 cand[kCand];
  u64 sorted[kCand];
  u64 warp_mass[kWarps], warp_best[kWarps];
  uint32_t warp_cnt[kWarps];
  // every CTA's largest key, tokens sent to the list and kept mass, in every CTA
  u64 best_of[kMaxCluster], mass_of[kMaxCluster];
  int sent_of[kMaxCluster];
  int n_cand;       // rank 0
  // a pass's result, written to every CTA by rank 0
  int bin;
  uint32_t bin_cnt, above_cnt, total_cnt;
  int sent;  // tokens of this CTA for the list
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
  double octaves;      // 256 log2(e) / T: (x - top) in 256ths of an octave
  double scale;        // mass of w = 1
  int mass_bits;       // its power of two
  const double *table;

  __device__ __forceinline__ void set(float top_, float temperature, int bits, const double *t) {
    top = top_;
    octaves = 369.3299304675746 / (double)temperature;
    mass_bits = bits;
    scale = (double)(1ull << bits);
    table = t;
  }
  // w of a logit that is not NaN, to 2^-42: with y = 256 log2 w split into an
  // integer k and |f| <= 1/2, w = 2^(k >> 8) 2^((k & 255) / 256) e^r for
  // r = f ln2 / 256, e^r by its series to r^3 (r^4 / 24 < 2^-42).  (Table look-up and
  // a short series: P. T. P. Tang, ACM TOMS 15(2), 1989.)
  __device__ __forceinline__ double w(float x) const { return w_scaled(x, 0); }
  // w 2^bits
  __device__ __forceinline__ double w_scaled(float x, int bits) const {
    if (top == INFINITY) return x == INFINITY ? (bits ? scale : 1.0) : 0.0;
    if (x == -INFINITY) return 0.0;
    constexpr double kMagic = 6755399441055744.0;  // 1.5 2^52: the sum's low word is round(y)
    constexpr double kC = 0.0027076061740622863;   // ln2 / 256
    const double y = fmax(((double)x - (double)top) * octaves, -240000.0);  // below: no mass
    const double kd = y + kMagic;
    const int k = __double2loint(kd);
    const double f = y - (kd - kMagic);
    double e = fma(f, kC * kC * kC / 6, kC * kC / 2);
    e = fma(f, e, kC);
    e *= f;
    const double t = table[k & 255];
    const double v = fma(t, e, t);
    return __hiloint2double(__double2hiint(v) + (((k >> 8) + bits) << 20), __double2loint(v));
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

// the bin of a logit that is not NaN, `top` the largest: rising as the logit falls
__device__ __forceinline__ int value_bin(float v, float top, float scale) {
  if (v == top) return 0;
  return (int)fminf((top - v) * scale, (float)(kBins - 1));
}

struct Row {
  cg::cluster_group cl;
  Shared &s;
  const float *x;  // the slice: shared memory, or the row in global memory
  int base, len;   // the slice's first token and length
  int rank, ctas;

  // whether token i of the slice, of logit v, is at or above a cut in the row's order
  __device__ __forceinline__ bool keeps(float v, int i, u64 cut) const {
    const float c = cut == kAll ? -INFINITY : order_value((uint32_t)(cut >> 32));
    return v > c || (v == c && token_key(v, base + i) >= cut);
  }
  template <class F>
  __device__ __forceinline__ void each(F f) {
    int i = threadIdx.x;
    for (; i + (kAhead - 1) * kThreads < len; i += kAhead * kThreads) {
      float v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) v[k] = x[i + k * kThreads];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) f(v[k], i + k * kThreads);
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

  // The first of the given bins at which the running count reaches k (k > 0) or the
  // running mass (k == 0) the target; see find().  The result lands in this CTA's s.bin
  // and beside it.
  __device__ void locate(const uint32_t *cnt, const u64 *mass, uint32_t k, float top_p,
                         uint32_t first_cnt, u64 first_mass) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kPer = kBins / kThreads;
    uint32_t c[kPer], csum = 0;
    u64 m[kPer], msum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      c[i] = cnt[threadIdx.x * kPer + i];
      m[i] = mass ? mass[threadIdx.x * kPer + i] : 0;
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
    if (threadIdx.x == kThreads - 1) s.total_cnt = cb + csum;
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
      locate(s.g_cnt, s.g_mass, k, top_p, first_cnt, first_mass);
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

  // The slice's tokens with keys >= within into the bins.  The last bin also takes all
  // that lies below the range: summed in registers first, as half the row may fall
  // there.
  template <class M>
  __device__ __forceinline__ void fill_bins(u64 within, float top, float scale, M mass) {
    uint32_t rest_n = 0;
    u64 rest_m = 0;
    each([&](float v, int i) {
      if (!keeps(v, i, within)) return;
      const u64 m = mass(v);
      const int bin = value_bin(v, top, scale);
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

  // the bins of one value per thread (NaN: none)
  __device__ __forceinline__ void fill_bins_with(float v, float top, float scale) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.cnt[i] = 0;
    __syncthreads();
    if (v == v) atomicAdd(&s.cnt[value_bin(v, top, scale)], 1u);
    __syncthreads();
  }

  // For a short top-k: the slice's first k tokens, and few more, into rank 0's list,
  // their number into s.sent.  The k-th largest of the threads' own maxima is not above
  // the slice's k-th largest, and few other tokens exceed it: so its bin, found among
  // one value per thread, bounds what is sent.  `mine`: this thread's maximum (NaN: no
  // token), `top`: the slice's.
  __device__ void send_first(uint32_t k, float mine, float top, float scale) {
    fill_bins_with(mine, top, scale);
    locate(s.cnt, nullptr, k, NAN, 0, 0);
    const int last = s.bin < 0 ? kBins - 1 : s.bin;
    auto sends = [&](float v) {
      return v == top || (top - v) * scale < (float)(last + 1) || (last == kBins - 1 && v == v);
    };
    each([&](float v, int i) {  // first into a list of this CTA's own
      if (!sends(v)) return;
      const int at = atomicAdd(&s.sent, 1);
      if (at < kCand) s.sorted[at] = token_key(v, base + i);
    });
    __syncthreads();
    if (ctas > 1) cl.barrier_wait();  // the row's CTAs have started
    const int n = s.sent;
    if (n > kCand) return;
    if (threadIdx.x == 0) s.bin = atomicAdd(cl.map_shared_rank(&s.n_cand, 0), n);
    __syncthreads();
    const int at = s.bin + threadIdx.x;
    if (threadIdx.x < n && at < kCand)
      *cl.map_shared_rank(&s.cand[at], 0) = s.sorted[threadIdx.x];
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

  // rank 0: the list in order of falling keys into s.sorted: a short one by counting
  // larger keys, else a bitonic sort, a key per thread, by shuffles within a warp and
  // through shared memory across warps.
  __device__ void sort_list(int n) {
    const int i = threadIdx.x;
    u64 key = i < n ? s.cand[i] : 0;
    if (n <= 128) {
      int place = 0;
      if (i < n)
#pragma unroll 4
        for (int j = 0; j < n; ++j) place += s.cand[j] > key;
      if (i < n) s.sorted[place] = key;
      __syncthreads();
      return;
    }
    int size = 32;
    while (size < n) size *= 2;
    for (int k = 2; k <= size; k *= 2) {
      for (int j = k / 2; j > 0; j /= 2) {
        u64 other;
        if (j >= 32) {
          if (i < size) s.sorted[i] = key;
          __syncthreads();
          other = i < size ? s.sorted[i ^ j] : 0;
          __syncthreads();
        } else {
          other = __shfl_xor_sync(0xffffffffu, key, j);
        }
        // falling runs where bit k of the index is 0
        const bool larger = ((i & k) == 0) == ((i & j) == 0);
        key = larger ? max(key, other) : min(key, other);
      }
    }
    if (i < size) s.sorted[i] = key;
    __syncthreads();
  }

  // The cut of the first k tokens (k > 0) or of the shortest prefix that holds
  // the top_p share of the mass, among the keys >= `within`: every CTA
  // returns the key of the last kept token.  Where `listed` is given and the tokens
  // down to the cut's bin fit the list, they are left there instead (*listed set).
  __device__ u64 cut(uint32_t k, float top_p, u64 within, const Weights &W, float bin_scale,
                     bool *listed) {
    clear_bins(!k);
    fill_bins(within, W.top, bin_scale, [&](float v) { return k ? 0 : W.mass(v); });
    find(k, top_p, 0, 0);
    if (s.bin < 0) return within;  // fewer than k tokens: all of them
    const int vbin = s.bin;
    if (listed && s.above_cnt + s.bin_cnt <= kCand) {
      *listed = true;
      gather([&](float v, u64 key) {
        return key >= within && value_bin(v, W.top, bin_scale) <= vbin;
      });
      return within;
    }
    // narrow a crowded bin by digits of the key, highest first
    int shift = 64, bits = 0;
    u64 prefix = 0;
    auto inside = [&](float v, u64 key) {
      return key >= within && value_bin(v, W.top, bin_scale) == vbin &&
             (shift == 64 || (key >> shift) == prefix);
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
      sort_list(n);
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
                              const Weights &W, float bin_scale, int32_t *token, float *prob) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = threadIdx.x;
    int n = s.n_cand;
    if (k && n > 128) {  // slices' lists joined: down to the bin of the k-th
      const u64 key = i < n ? s.cand[i] : 0;
      const float v = i < n ? order_value((uint32_t)(key >> 32)) : NAN;
      fill_bins_with(v, W.top, bin_scale);
      locate(s.cnt, nullptr, k, NAN, 0, 0);
      if (threadIdx.x == 0) s.n_cand = 0;
      __syncthreads();
      if (i < n && (s.bin < 0 || value_bin(v, W.top, bin_scale) <= s.bin))
        s.cand[atomicAdd(&s.n_cand, 1)] = key;
      __syncthreads();
      n = s.n_cand;
    }
    sort_list(n);
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
    sort_list(n_keep);
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
    const mlm_sample_params *params, const float *uniform, const int32_t *step, int32_t *token,
    float *prob) {
  extern __shared__ __align__(16) uint8_t s_raw[];
  Shared &s = *reinterpret_cast<Shared *>(s_raw);
  float *s_x = reinterpret_cast<float *>(s_raw + sizeof(Shared));
  cg::cluster_group cl = cg::this_cluster();
  const int rank = cl.block_rank(), ctas = cl.num_blocks();
  if (threadIdx.x == 0) s.n_cand = s.sent = 0;
  if (threadIdx.x < 256) s.exp2_256[threadIdx.x] = exp2(threadIdx.x / 256.0);
  pdl_wait_then_release();
  __syncthreads();
  if (ctas > 1) cl.barrier_arrive();
  const int row = blockIdx.x / ctas;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int base = min(n, rank * slice), len = min(n - base, slice);
  const float *g = logits + row * row_stride + base;
  const mlm_sample_params p = params[row];
  Row r{cl, s, g, base, len, rank, ctas};

  // the slice into shared memory; its largest logit, the first of equals
  float mine = -INFINITY;
  int mine_at = -1;
  r.each([&](float v, int i) {
    if (resident) s_x[i] = v;
    if (v > mine) {
      mine = v;
      mine_at = i;
    }
  });
  if (resident) r.x = s_x;
  u64 best = mine_at < 0 ? 0 : token_key(mine, base + mine_at);
  {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
    if (lane == 0) s.warp_best[warp] = ((u64)hi << 32) | lo;
  }
  __syncthreads();
  best = s.warp_best[lane];
  {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
    best = ((u64)hi << 32) | lo;
  }
  if (best < kAll) {  // nothing above -inf: the first -inf, if there is one
    uint32_t first = 0;
    r.each([&](float v, int i) {
      if (v == -INFINITY) first = max(first, ~(uint32_t)(base + i));
    });
    first = __reduce_max_sync(0xffffffffu, first);
    __syncthreads();
    if (lane == 0) s.warp_best[warp] = first;
    __syncthreads();
    first = __reduce_max_sync(0xffffffffu, (uint32_t)s.warp_best[lane]);
    best = first ? ((u64)order_bits(-INFINITY) << 32) | first : 0;
  }

  // bins over the logits that matter: 24 temperatures, but at least 16 and at
  // most 64 below the largest
  const float bin_scale = (float)kBins / fminf(fmaxf(24.f * p.temperature, 16.f), 64.f);
  const uint32_t k = p.top_k > 0 && p.top_k < n ? (uint32_t)p.top_k : 0;
  // half the list for the slices' first k, the rest for what shares their last bins
  const bool is_short = k && 2 * (u64)k * ctas <= kCand && p.temperature > 0.f;
  if (is_short && best >= kAll)
    r.send_first(k, mine_at < 0 ? NAN : mine, order_value((uint32_t)(best >> 32)), bin_scale);
  else if (ctas > 1)
    cl.barrier_wait();
  int sent = 0;
  if (ctas > 1) {
    __syncthreads();
    if (threadIdx.x < ctas) {
      Shared *o = cl.map_shared_rank(&s, threadIdx.x);
      o->best_of[rank] = best;
      o->sent_of[rank] = s.sent;
    }
    cl.sync();
    best = s.best_of[lane < ctas ? lane : 0];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    sent = __reduce_add_sync(0xffffffffu, lane < ctas ? s.sent_of[lane] : 0);
  } else {
    __syncthreads();
    sent = s.sent;
  }

  const float top = order_value((uint32_t)(best >> 32));
  const bool none = best < kAll || top == -INFINITY;
  if (none || !(p.temperature > 0.f)) {
    if (rank == 0 && threadIdx.x == 0) {
      // only NaN: 0, as the argmax
      token[row] = best < kAll ? 0 : (int32_t)~(uint32_t)best;
      if (prob) prob[row] = none ? 0.f : 1.f;
    }
    return;
  }
  Weights W;
  W.set(top, p.temperature, mass_bits, s.exp2_256);
  const double min_w = p.min_p > 0.f ? fmin((double)p.min_p, 1.0) : 0.0;
  // step: rows of uniforms per step of a replayed graph
  float u = uniform[(step ? (size_t)*step * (gridDim.x / ctas) : 0) + row];
  u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;  // NaN: 0
  u64 cut = kAll;
  bool listed = is_short && sent <= kCand;
  if (k && !listed) cut = r.cut(k, NAN, cut, W, bin_scale, &listed);
  if (p.top_p < 1.f && !listed) cut = r.cut(0, p.top_p, cut, W, bin_scale, k ? nullptr : &listed);
  if (listed) {
    if (rank == 0)
      r.draw_listed(k, p.top_p, k ? 0 : s.target, min_w, u, W, bin_scale, token + row,
                    prob ? prob + row : nullptr);
    return;  // nothing of this CTA's shared memory is read any more
  }

  // the kept mass of every warp's stretch
  auto kept = [&](float v, int i) -> u64 {
    if (!r.keeps(v, i, cut)) return 0;
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
    if (threadIdx.x < ctas) cl.map_shared_rank(&s, threadIdx.x)->mass_of[rank] = total;
    cl.sync();
    const u64 of = lane < ctas ? s.mass_of[lane] : 0;
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
}

constexpr int kMaxN = 1 << 22;
// shared memory a slice may take beside the bins (one CTA per SM)
constexpr size_t kSliceBytes = 150 * 1024;
static_assert(sizeof(Shared) + kSliceBytes <= 227 * 1024, "a CTA's shared memory");

}  // namespace

int sample_init(mlm_ctx *ctx) {
  MLM_CUDA_TRY(ctx, cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)(sizeof(Shared) + kSliceBytes)));
  return MLM_OK;
}

int sample_launch(mlm_ctx *ctx, const float *logits, int rows, int n, int64_t row_stride,
                  const mlm_sample_params *params, const float *uniform, const int32_t *step,
                  int32_t *token, float *prob, cudaStream_t stream) {
  int ctas = kMaxCluster;
  // twice the SMs' number of CTAs: rows of different settings take different times
  while (ctas > 1 && (rows * ctas > 2 * ctx->sm_count || n < kMinSlice * ctas)) ctas /= 2;
  const int slice = (n + ctas - 1) / ctas;
  const int resident = (size_t)slice * 4 <= kSliceBytes;
  int bits = 62;
  while ((1ll << (62 - bits)) < n) --bits;
  bits = std::min(bits, 50);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared) + (resident ? (size_t)slice * 4 : 0);
  cfg.stream = stream;
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
                                             slice, resident, bits, params, uniform, step, token,
                                             prob),
                          "mlm_sample_f32");
}

int sample_max_n() { return kMaxN; }

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
  return sample_launch(ctx, logits, rows, n, row_stride, params, uniform, nullptr, token, prob,
                       ctx->stream);
}
