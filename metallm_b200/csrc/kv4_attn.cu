// kv4_attn.cu -- grouped-query attention over the 4-bit KV cache.
//
// out = softmax(q K^T / sqrt(128)) V for every new token of every sequence, K
// and V the values m + d c the cache rows stand for (the fp16 cache's
// counterpart is mlm_attn_decode; LlamaRunner.swift:669-952).
//
// Up to 16 (token, head) rows per KV head here; more in kv4_attn_many.cu.
#include <algorithm>
#include <type_traits>

#include "kv4_common.cuh"
#include "q4k_gemv_common.cuh"

namespace mlm {
namespace {

constexpr int kRow = kKv4Row;
constexpr int kD = kKv4D;

// ---------------------------------------------------------------------------
// Few rows: up to 16 (token, head) pairs of one KV head at once -- a decode
// step, a few drafted tokens.  The floor is the cache's bytes (160 per position
// and KV head).
//
// Both products run on the tensor cores on the codes themselves.  A masked
// nibble in a binary16's low mantissa bits is the subnormal c 2^-24 (16 c
// 2^-24 one nibble up), so one AND makes two operands; the group's d and m,
// constant along the 32 elements of a group, enter outside the product:
//   q.k = sum_g d_g (sum_i q_i c_i) + m_g (sum_i q_i)
//   o_i = sum_j (p_j d_jg) c_ji + sum_j p_j m_jg
// K is the A operand (16 rows x 16 dimensions), the queries the 8 columns of
// B; V^T is the A operand (16 dimensions x 16 rows; ldmatrix.trans of the codes
// as 16-bit units hands a lane the nibbles of two neighbouring rows side by
// side), the weights p d the 8 columns of B.  Nothing of K or V is rounded; q is
// fp16 already (scaled by a power of two per row, so that q / 16 stays exact).  For an
// fp16 output p and p d go in as fp16 hi + lo, and with at most four columns the hi and
// lo parts share the eight columns of one product; for a bf16 output p is rounded to fp16
// and p d once more.  Scores, statistics and sums are fp32.
//
// Work is cut by bytes, not by head: the blocks of 32 rows of every (sequence,
// KV head) form one line, cut into equal stretches per CTA and again per warp
// from the lengths in device memory, so ragged batches and graph replays stay
// balanced.  A warp streams its blocks through a ring of its own (two 2560-byte
// bulk copies per block, contiguous in the cache) and keeps a running maximum
// and sum per column.  Stretches of one head are joined in order: a warp's
// pieces by their CTA, the CTAs' through the context's scratch by the last CTA of the
// head to arrive, so sums do not depend on timing.
//
// Measured: 64 sequences x 8192 rows x 8 KV heads (673 MB) 117 us, 5.75 TB/s (139 us once
// a second of such calls has the card at its power limit, 1660 MHz for 1965); 131071 rows
// x 8 (168 MB) 45 us; 2048 rows 10 us, some 5 us of it the cut, the first copies and the
// joins.  On 24 ragged sequences no unit is full: issue slots 60 %, the ALU pipe (masks,
// transposes, conversions) 53 %, DRAM 48 %; 718 instructions per block of 32 rows in four
// warps per scheduler, each a chain from the copy to the second product.  128 registers
// hold the body of 8 columns but for 32 to 40 bytes.  Sixteen columns take 1350
// instructions per block in two warps per scheduler, issue slots 32 %: 8 x 4 tokens at
// 4099 rows 39 us.  Warps, ring: 16 x 2 stages for 8 columns, 8 x 4 for 16 (the reverse:
// 139 us for the 64 sequences, 58 against 38 us for 8 x 4 tokens).
// ---------------------------------------------------------------------------

constexpr int kBlk = 32;                     // cache rows per block
constexpr int kHalfStage = kBlk * kRow;      // K or V of a block
constexpr int kStage = 2 * kHalfStage;
constexpr int kPieceRow = kD + 4;            // a column of a piece: o[128], m, l, padding
constexpr int kMaxCols = 16;
// Weights are 2^(s - max + kBias), a score at most 2^kLead above the maximum, so p is below
// 2^14; d goes in scaled by a power of two per group that brings the largest of the item so
// far into [1, 2), so p d is below 2^15.  Both are then held to 2^-25, 2^-35 of the largest
// weight (times the largest scale), which is what the many small weights behind a large one
// need: 2^17 rows add up to 2^-18 at most that way.
constexpr float kLead = 4.f, kBias = 10.f;

// a product from zero accumulators
__device__ __forceinline__ void mma_f16_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                             uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// a += b.  A product's accumulators are cut off, not rounded: left in them over a long
// stretch the codes' and the minima's parts of an output, which nearly cancel, shrink by
// some 2^-24 of themselves per product (16 sequences of 131072 rows: an error of 4.5e-3 of
// the norm, 1.7e-3 with a block's products from zero and added here).
__device__ __forceinline__ void add4(float (&a)[4], const float (&b)[4]) {
#pragma unroll
  for (int i = 0; i < 4; i += 2)
    asm("{\n .reg .b64 x, y;\n mov.b64 x, {%0, %1};\n mov.b64 y, {%2, %3};\n"
        " add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
        : "+f"(a[i]), "+f"(a[i + 1])
        : "f"(b[i]), "f"(b[i + 1]));
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void ldsm2_t(uint32_t addr, uint32_t (&r)[2]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
               : "=r"(r[0]), "=r"(r[1])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t lds4(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
// the transpose of an 8x8 matrix of 16-bit elements, row r of it in lanes 4r ..
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// (the cache is read once per step: evict-first, so that it does not push the kernel's
// code and the partial sums out of L2)
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void *src, uint32_t bytes,
                                          uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1], %2, [%3], %4;" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b),
                            *reinterpret_cast<const __half2 *>(&c));
  return *reinterpret_cast<const uint32_t *>(&r);
}

// The four nibbles of each 16-bit half as subnormal binary16 values, a power of two each
// (code_unit) times the code.  A product's terms are aligned by their operands' exponents,
// which are all that of the largest subnormal, and cut off below some 2^-24 of the largest
// term's: a code k bits below the top loses k bits, always downwards, and a sum over a long
// cache nearly cancels with its m part.  In place (bits 0 and 4) that cost an fp16 output of
// 60001 rows 5e-4 of its norm, against 2.1e-4 for its rounding.  So all four come to bit 4
// for it (three shifts, 64 x 8192 rows 120.8 us); for a bf16 output, whose rounding is eight
// times coarser, one shift takes two of them to bits 2 and 6 (115.8 us, 112.8 in place).
template <bool EXACT>
__device__ __forceinline__ void spread_codes(uint32_t w, uint32_t (&v)[4]) {
  if (EXACT) {
    v[0] = (w << 4) & 0x00F000F0u;
    v[1] = w & 0x00F000F0u;
    v[2] = (w >> 4) & 0x00F000F0u;
    v[3] = (w >> 8) & 0x00F000F0u;
  } else {
    v[0] = (w << 2) & 0x003C003Cu;
    v[1] = (w << 2) & 0x03C003C0u;
    v[2] = (w >> 6) & 0x003C003Cu;
    v[3] = (w >> 6) & 0x03C003C0u;
  }
}
// 2^24 over the factor of nibble i
template <bool EXACT>
__device__ __forceinline__ float code_unit(int i) {
  return EXACT ? 1048576.f : (i & 1) ? 262144.f : 4194304.f;
}

// The unit 2^e, -15 <= e <= 15, that V's scales of a group are counted in: its reciprocal,
// a binary16 value twice, by which they are multiplied
__device__ __forceinline__ uint32_t unit_of(int e) {
  return (e < 15 ? (uint32_t)(15 - e) << 10 : 0x0200u) * 0x10001u;
}
__device__ __forceinline__ int unit_exponent(uint32_t unit) { return 15 - (int)((unit & 0xFFFFu) >> 10); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// an item (the blocks of one KV head of one sequence) and a block of it
struct Item {
  int b, h, blk, nb;
  int len, count;  // of sequence b
};

// Joins the parts of an item that CTAs c0 .. c1 share, in order: a warp per column and
// 32 V dimensions, whose parts' loads are in flight together.
template <int V, class OutT>
__device__ __forceinline__ void join_parts(const Kv4AttnArgs &a, const Item &of, int c0, int c1,
                                           int warp, int warps) {
  static_assert(V == 2 || V == 4, "one load per part");
  constexpr int kTasks = 4 / V;  // per column
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int t = warp; t < kTasks * of.count * a.group; t += warps) {
    const int col = t / kTasks, d = (t % kTasks) * 32 * V + V * lane;
    auto part_of = [&](int c) {
      return a.parts + (((size_t)c * 2 + (c == c0 ? 1 : 0)) * kMaxCols + col) * kPieceRow;
    };
    float top = -INFINITY, sum = 0.f, v[V] = {};
    // 32 parts at a time, their statistics one per lane; a new maximum rescales
#pragma unroll 1
    for (int cb = c0; cb <= c1; cb += 32) {
      const int n = min(32, c1 - cb + 1);
      const bool in = lane < n;
      const float2 ml = __ldcg(reinterpret_cast<const float2 *>(part_of(cb + (in ? lane : 0)) + kD));
      const float m = in ? ml.x : -INFINITY;
      const float up = fmaxf(top, warp_max(m));
      const float old = top == up ? 1.f : ex2(top - up), f = m == up ? 1.f : ex2(m - up);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] *= old;
      sum = sum * old + (in ? f * ml.y : 0.f);
      top = up;
#pragma unroll 1
      for (int k0 = 0; k0 < n; k0 += 8) {
        float w[8][V];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float *p = part_of(min(cb + k0 + k, c1)) + d;
          if (V == 4) {
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(p));
            w[k][0] = x.x, w[k][1] = x.y, w[k][V - 2] = x.z, w[k][V - 1] = x.w;
          } else {
            const float2 x = __ldcg(reinterpret_cast<const float2 *>(p));
            w[k][0] = x.x, w[k][1] = x.y;
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float fk = __shfl_sync(0xffffffffu, f, (k0 + k) & 31);
          if (k0 + k < n)
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = fmaf(fk, w[k][i], v[i]);
        }
      }
    }
    sum = warp_sum(sum);
    const int tok = a.tokens == 1 ? 0 : col / a.group;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    OutT *dst = reinterpret_cast<OutT *>(a.out) +
                (((size_t)of.b * a.tokens + tok) * a.n_heads + of.h * a.group + (col - tok * a.group)) * kD + d;
    OutT e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_float<OutT>(v[i] * inv);
#pragma unroll
    for (int i = 0; i < V; i += 2)
      *reinterpret_cast<uint32_t *>(dst + i) = *reinterpret_cast<const uint32_t *>(e + i);
  }
}

template <int NT, bool DUP, int W, int STAGES, class OutT>
__global__ void __launch_bounds__(W * 32, 1) kv4_attn_few_kernel(Kv4AttnArgs a) {
  static_assert(2 * W <= 32, "a lane per piece");
  static_assert(!DUP || NT == 1, "hi and lo share one tile of columns");
  constexpr int kCols = DUP ? 4 : 8 * NT;
  constexpr int kPiece = kCols * kPieceRow;
  // An fp16 output takes the weights as hi + lo (rounded to fp16 alone they would
  // add as much error as the output's own rounding, as codes are not centred);
  // for a bf16 output, eight times coarser, hi alone
  constexpr bool LO = std::is_same<OutT, __half>::value;
  constexpr bool kSplit = DUP && LO;  // columns 4 .. 7 hold the lo parts
  static_assert(kPiece * 4 <= STAGES * kStage, "a warp's last piece lies in its ring");
  extern __shared__ __align__(128) uint8_t smem[];
  // rings, the line's offsets per sequence
  int *s_off = reinterpret_cast<int *>(smem + W * STAGES * kStage);  // [batch + 1]
  __shared__ __align__(8) uint64_t s_bar[W][STAGES];
  __shared__ int s_item[2 * W];  // pieces: the item's first block (-1: none)
  __shared__ Item s_of[2 * W];   // and the item
  __shared__ bool s_last[2];
  // per warp, out of the registers: the item at hand and the one being copied
  __shared__ Item s_cur[W], s_ahead[W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = lane >> 2, t4 = lane & 3;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * STAGES * kStage;
  const uint32_t bar0 = (uint32_t)__cvta_generic_to_shared(&s_bar[warp][0]);
  if (lane == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(bar0 + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x < 2 * W) s_item[threadIdx.x] = -1;
  pdl_wait_then_release();

  // the line's offsets: sequence b's blocks start at s_off[b]
  if (warp == 0) {
    int run = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
      const int b = b0 + lane;
      int n = 0;
      if (b < a.batch) {
        int len, count;
        seq_shape(a, b, len, count);
        n = count > 0 ? (len + kBlk - 1) / kBlk * a.n_kv : 0;
        if (blockIdx.x == 0 && seq_outside(a, b)) report_outside(a.status);
      }
      int in = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, in, o);
        if (lane >= o) in += up;
      }
      if (b < a.batch) s_off[b] = run + in - n;
      run += __shfl_sync(0xffffffffu, in, 31);
    }
    if (lane == 0) s_off[a.batch] = run;
  }
  __syncthreads();
  const int total = s_off[a.batch];
  // tokens that attend to nothing in sequences without blocks
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    if (s_off[b + 1] > s_off[b]) continue;
    int len, count;
    seq_shape(a, b, len, count);
    OutT *o = reinterpret_cast<OutT *>(a.out) + (size_t)b * a.tokens * a.n_heads * kD;
    for (int i = threadIdx.x; i < count * a.n_heads * kD; i += W * 32) o[i] = from_float<OutT>(0.f);
  }
  // equal stretches; a CTA with few blocks gives them to its first warps, one
  // per SM quarter
  const int quota = max(4, (total + (int)gridDim.x - 1) / (int)gridDim.x);
  const int cta0 = min(total, (int)blockIdx.x * quota), cta1 = min(total, cta0 + quota);
  if (cta0 >= cta1) return;
  const int per = (cta1 - cta0) / W, more = (cta1 - cta0) % W;
  const int w0 = cta0 + warp * per + min(warp, more), w1 = w0 + per + (warp < more ? 1 : 0);

  auto at = [&](int x) {
    int lo = 0, hi = a.batch;  // the last b with s_off[b] <= x
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_off[mid] <= x) lo = mid; else hi = mid;
    }
    Item c;
    c.b = lo;
    seq_shape(a, lo, c.len, c.count);
    c.nb = (c.len + kBlk - 1) / kBlk;
    const int rem = x - s_off[lo];
    c.h = rem / c.nb;
    c.blk = rem - c.h * c.nb;
    return c;
  };
  auto next_item = [&](Item &c) {
    c.blk = 0;
    if (++c.h < a.n_kv) return;
    c.h = 0;
    do ++c.b; while (c.b < a.batch && s_off[c.b + 1] == s_off[c.b]);
    if (c.b == a.batch) return;
    seq_shape(a, c.b, c.len, c.count);
    c.nb = (c.len + kBlk - 1) / kBlk;
  };
  auto source = [&](const Item &c) {
    return a.kc + (((size_t)c.b * a.n_kv + c.h) * a.capacity + (size_t)c.blk * kBlk) * kRow;
  };
  const uint8_t *src = nullptr;  // the next block to copy
  const long long k_to_v = a.vc - a.kc;
  int to_copy = w1 - w0, rows_ahead = 0;  // blocks of this stretch, rows of the item, to come
  int blk = 0;                            // of the item at hand
  auto keep = [&](Item &slot, const Item &c) {
    __syncwarp();
    if (lane == 0) slot = c;
    __syncwarp();
  };
  if (to_copy > 0) {
    const Item c = at(w0);
    keep(s_cur[warp], c);
    keep(s_ahead[warp], c);
    src = source(c);
    rows_ahead = c.len - c.blk * kBlk;
    blk = c.blk;
  }
  // copy the next block into a stage and move on
  auto copy = [&](int stage) {
    if (lane == 0) {
      const uint32_t bytes = (uint32_t)min(kBlk, rows_ahead) * kRow;
      const uint32_t bar = bar0 + 8 * stage, dst = ring + stage * kStage;
      mbar_expect_tx(bar, 2 * bytes);
      const uint64_t policy = evict_first_policy();
      bulk_copy(dst, src, bytes, bar, policy);
      bulk_copy(dst + kHalfStage, src + k_to_v, bytes, bar, policy);
    }
    --to_copy;
    src += kHalfStage;
    rows_ahead -= kBlk;
    if (rows_ahead <= 0 && to_copy > 0) {
      Item c = s_ahead[warp];
      next_item(c);
      keep(s_ahead[warp], c);
      src = source(c);
      rows_ahead = c.len;
    }
  };
  // the first item's queries into L1, ahead of the copies that would keep them waiting:
  // two lines per column
  if (to_copy > 0) {
    const Item c = s_cur[warp];
    const int col = lane >> 1, tok = a.tokens == 1 ? 0 : col / a.group;
    if (col < c.count * a.group)
      asm volatile("prefetch.global.L1 [%0];" ::"l"(
          a.q + (((size_t)c.b * a.tokens + tok) * a.n_heads + c.h * a.group + (col - tok * a.group)) * kD +
          64 * (lane & 1)));
  }
#pragma unroll
  for (int i = 0; i < STAGES; ++i)
    if (to_copy > 0) copy(i);

  // Pieces that end within a warp's stretch wait in the scratch (the ring is in use);
  // the stretch's last one lies in the ring
  float *heads = a.parts + (size_t)2 * gridDim.x * kMaxCols * kPieceRow + (size_t)blockIdx.x * W * kPiece;

  const bool lo_lane = kSplit && r >= 4;  // with shared columns: this lane's part

  // queries: the B operand of K's products, per group of 32 dimensions
  uint32_t qb[NT][4][4];
  float cs[NT];                // score scale of column r, in powers of two
  int seen[NT];                // rows column r attends to
  uint32_t qm[NT][2];          // the B operand of K's minima: (0, group sum) per group, hi and lo
  float o[NT][4][2][4], mx[NT], l[NT];
  uint32_t unit = 0;           // even r: what V's scales of group r / 2 are multiplied by, twice
  float om[NT][4];             // sum of p m: rows 2 g + 1 of the product with V's scales
  bool ok = true;
  int stage = 0;
  uint32_t phase = 0;

  for (int x = w0; x < w1;) {
    const int first_blk = blk;
    const int end_blk = min(s_cur[warp].nb, blk + w1 - x);  // this stretch's part of the item
    x += end_blk - first_blk;
    int mask_from;  // the first block with a row that some token does not see
    {
      const Item cur = s_cur[warp];
      const int len = cur.len, count = cur.count;
      mask_from = max(0, len - count + 1) / kBlk;
      unit = r & 1 ? 0x3C003C00u : 0x78007800u;  // 1, and 2^15 until the first block's scales are known
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int col = DUP ? (r & 3) : nt * 8 + r;
        const bool live = col < count * a.group;
        const int tok = live && a.tokens > 1 ? col / a.group : 0;
        seen[nt] = live ? max(0, len - count + tok + 1) : 0;
        const __half *qr = a.q + (((size_t)cur.b * a.tokens + tok) * a.n_heads +
                                  cur.h * a.group + (col - tok * a.group)) * kD + 8 * t4;
        float f[4][8], big = 0.f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const uint4 v = live ? *reinterpret_cast<const uint4 *>(qr + 32 * g) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 p = unpack_f16(u4_get(v, i));
            f[g][2 * i] = p.x;
            f[g][2 * i + 1] = p.y;
            big = fmaxf(big, fmaxf(fabsf(p.x), fabsf(p.y)));
          }
        }
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        // the largest |q| of the row into [2^13, 2^14): q / 16 keeps its bits (an infinite one
        // as the largest finite, so that cs stays a positive number)
        big = fminf(big, 65504.f);
        const int e = big > 0.f ? 13 - ((int)((__float_as_uint(big) >> 23) & 0xFF) - 127) : 0;
        const float up = __uint_as_float((uint32_t)(e + 127) << 23);
        cs[nt] = kInvSqrtD * kLog2e * __uint_as_float((uint32_t)(24 - e + 127) << 23);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            f[g][i] *= up;
            sum += f[g][i];
          }
          qb[nt][g][0] = pack_f16(f[g][0], f[g][4]);
          qb[nt][g][1] = pack_f16(f[g][1] * 0.0625f, f[g][5] * 0.0625f);
          qb[nt][g][2] = pack_f16(f[g][2], f[g][6]);
          qb[nt][g][3] = pack_f16(f[g][3] * 0.0625f, f[g][7] * 0.0625f);
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          sum *= 0.015625f;  // at most 32 x 2^14: below 2^13
          const float hi = __half2float(__float2half_rn(sum));
          if (t4 == g) {
            qm[nt][0] = pack_f16(0.f, hi);
            qm[nt][1] = pack_f16(0.f, sum - hi);
          }
          om[nt][g] = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) o[nt][g][0][i] = o[nt][g][1][i] = 0.f;
        }
        mx[nt] = -INFINITY;
        l[nt] = 0.f;
      }
    }
    auto block = [&](auto mask_tag) {
      constexpr bool MASK = decltype(mask_tag)::value;
      const uint32_t sk = ring + stage * kStage, sv = sk + kHalfStage;
      const uint32_t tile_lane =
          (uint32_t)((((lane >> 3) & 1) * 8 + (lane & 7)) * kRow + (lane >> 4) * 16);
      // scores of the block's two 16-row tiles
      float sT[NT][2][2][2];  // column r: rows 16 kt + 8 half + 2 t4 + {0, 1}
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        uint32_t w[2][4];
        ldsm4(sk + kt * 16 * kRow + tile_lane, w[0]);
        ldsm4(sk + kt * 16 * kRow + tile_lane + 32, w[1]);
        const uint4 dm0 = lds16(sk + (kt * 16 + r) * kRow + 64);
        const uint4 dm1 = lds16(sk + (kt * 16 + r + 8) * kRow + 64);
        // sum_g m_g (sum q): the scale words (d, m) are an A operand already
        const uint32_t me0 = lds4(sk + (kt * 16 + r) * kRow + 64 + 4 * t4);
        const uint32_t me1 = lds4(sk + (kt * 16 + r + 8) * kRow + 64 + 4 * t4);
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float acc[4];
          mma_f16_zero(acc, me0, me1, me0, me1, qm[nt][0], qm[nt][1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[nt][i] = acc[i] * 3.814697265625e-06f;  // to units of 2^-24
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const uint32_t wa = w[g >> 1][(g & 1) * 2], wb = w[g >> 1][(g & 1) * 2 + 1];
          const uint32_t wa8 = wa >> 8, wb8 = wb >> 8;
          const float d0 = low_f16(u4_get(dm0, g)), d1 = low_f16(u4_get(dm1, g));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float acc[4];
            mma_f16_zero(acc, wa & 0x000F000Fu, wb & 0x000F000Fu, wa & 0x00F000F0u,
                         wb & 0x00F000F0u, qb[nt][g][0], qb[nt][g][1]);
            mma_f16_16816(acc, wa8 & 0x000F000Fu, wb8 & 0x000F000Fu, wa8 & 0x00F000F0u,
                          wb8 & 0x00F000F0u, qb[nt][g][2], qb[nt][g][3]);
            s[nt][0] = fmaf(d0, acc[0], s[nt][0]);
            s[nt][1] = fmaf(d0, acc[1], s[nt][1]);
            s[nt][2] = fmaf(d1, acc[2], s[nt][2]);
            s[nt][3] = fmaf(d1, acc[3], s[nt][3]);
          }
        }
        // rows x columns to columns x rows, as the V product's B operand wants
        // the weights: 32-bit values as two 16-bit matrices
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t v0 = __float_as_uint(s[nt][2 * half]),
                           v1 = __float_as_uint(s[nt][2 * half + 1]);
            const uint32_t lo = transpose8(__byte_perm(v0, v1, 0x5410));
            const uint32_t hi = transpose8(__byte_perm(v0, v1, 0x7632));
            sT[nt][kt][half][0] = __uint_as_float(__byte_perm(lo, hi, 0x5410));
            sT[nt][kt][half][1] = __uint_as_float(__byte_perm(lo, hi, 0x7632));
          }
      }
      // Rows that a column does not see get no weight.  A value row with NaN scales
      // (0 x NaN is not 0) or past the sequence goes in with zero scales; the NaN shows
      // in the weight of the columns that see it.
      uint32_t good = 0xFFu;
      if (MASK) {
        const int row0 = blk * kBlk + 2 * t4, len = s_cur[warp].len;
        good = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = (i >> 2) * 16 + ((i >> 1) & 1) * 8 + (i & 1);
          const uint4 dm = lds16(sv + (2 * t4 + at) * kRow + 64);
          const bool bad = not_finite(dm.x) || not_finite(dm.y) || not_finite(dm.z) || not_finite(dm.w);
          if (row0 + at < len && !bad) good |= 1u << i;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float &v = sT[nt][i >> 2][(i >> 1) & 1][i & 1];
            if (bad) v = NAN;
            if (row0 + at >= seen[nt]) v = -INFINITY;
          }
        }
      }
      auto good_pair = [&](int kt, int j) -> uint32_t {
        const uint32_t bits = good >> (4 * kt + 2 * j);
        return ((bits & 1) ? 0xFFFFu : 0u) | ((bits & 2) ? 0xFFFF0000u : 0u);
      };
      // V's transposed scale words: d in the lanes of even r, in the group's unit, m in the
      // others.  A scale of 2 units or more has bit 14 set
      uint32_t mt[2][2];
      auto value_scales = [&] {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          ldsm2_t(sv + (kt * 16 + (lane & 15)) * kRow + 64, mt[kt]);
          if (MASK) {
            mt[kt][0] &= good_pair(kt, 0);
            mt[kt][1] &= good_pair(kt, 1);
          }
        }
      };
      auto to_units = [&] {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int j = 0; j < 2; ++j) mt[kt][j] = hmul2(mt[kt][j], unit);
      };
      value_scales();
      to_units();
      const uint32_t any_d = mt[0][0] | mt[0][1] | mt[1][0] | mt[1][1];
      if (__any_sync(0xffffffffu, (any_d & (r & 1 ? 0u : 0x40004000u)) != 0)) {
        // larger scales than before (or infinities, NaN): larger units, what has been
        // summed scaled to them
        value_scales();
        uint32_t big = __vmaxu2(__vmaxu2(mt[0][0] & 0x7FFF7FFFu, mt[0][1] & 0x7FFF7FFFu),
                                __vmaxu2(mt[1][0] & 0x7FFF7FFFu, mt[1][1] & 0x7FFF7FFFu));
        big = max(big & 0xFFFFu, big >> 16);
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const int was = unit_exponent(unit);
        const int now = r & 1 ? was : max(was, min((int)(big >> 10) - 15, 15));
        unit = unit_of(now);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float f = power_of_two(__shfl_sync(0xffffffffu, was - now, 8 * g));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[nt][g][0][i] *= f, o[nt][g][1][i] *= f;
        }
        to_units();
      }
      // Running maximum and sum.  The maximum follows only when a score leads it
      // by more than 2^kLead; the factor is l's too.
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, sT[nt][i >> 2][(i >> 1) & 1][i & 1]);
        if (__any_sync(0xffffffffu, (top - mx[nt]) * cs[nt] > kLead)) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          top = fmaxf(top, mx[nt]);
          const float f = top == mx[nt] ? 1.f : ex2((mx[nt] - top) * cs[nt]);
          l[nt] *= f;
          const float f0 = __shfl_sync(0xffffffffu, f, 8 * t4),
                      f1 = __shfl_sync(0xffffffffu, f, 8 * t4 + 4);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            om[nt][g] *= (g & 1) ? f1 : f0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              o[nt][g][i][0] *= f0;
              o[nt][g][i][1] *= f1;
              o[nt][g][i][2] *= f0;
              o[nt][g][i][3] *= f1;
            }
          }
          mx[nt] = top;
        }
        const float base = fmaf(mx[nt] == -INFINITY ? 0.f : mx[nt], -cs[nt], kBias);
        float sum = 0.f;  // the block's first: thousands of equal weights one by one are rounded alike
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float &v = sT[nt][i >> 2][(i >> 1) & 1][i & 1];
          v = ex2(fmaf(v, cs[nt], base));
          sum = i == 0 ? v : sum + v;
        }
        l[nt] += sum;
      }
      // the weights of the lane's eight rows as fp16 hi (and lo) pairs, and the m part:
      // sum_j p_j m_jg (and p_j d_jg, unused)
      uint32_t ph[NT][2][2], pl[NT][2][2], pn[NT][2][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float sum[4];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float(&p)[2] = sT[nt][kt][j];
            uint32_t &h = ph[nt][kt][j], &lo = pl[nt][kt][j], &n = pn[nt][kt][j];
            h = pack_f16(p[0], p[1]);
            lo = n = 0;
            if (LO) {
              const float2 f = unpack_f16(h);
              lo = pack_f16(p[0] - f.x, p[1] - f.y);
              if (DUP) {
                lo = lo_lane ? lo : 0u;
                n = lo_lane ? h ^ 0x80008000u : 0u;
              }
            }
          }
          const uint32_t b0 = kSplit && lo_lane ? pl[nt][kt][0] : ph[nt][kt][0],
                         b1 = kSplit && lo_lane ? pl[nt][kt][1] : ph[nt][kt][1];
          if (kt == 0)
            mma_f16_zero(sum, mt[kt][0], 0u, mt[kt][1], 0u, b0, b1);
          else
            mma_f16_16816(sum, mt[kt][0], 0u, mt[kt][1], 0u, b0, b1);
          if (LO && !DUP) mma_f16_16816(sum, mt[kt][0], 0u, mt[kt][1], 0u, pl[nt][kt][0], pl[nt][kt][1]);
        }
        add4(om[nt], sum);
      }
      // o += (p d) c
#pragma unroll
      for (int gp = 0; gp < 2; ++gp) {
        uint32_t w[2][4];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) ldsm4_t(sv + kt * 16 * kRow + tile_lane + 32 * gp, w[kt]);
#pragma unroll
        for (int gi = 0; gi < 2; ++gi) {
          const int g = 2 * gp + gi;
          uint32_t bh[NT][2][2], bl[NT][2][2];
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              // d of rows 2 t4, + 1 (and of rows 2 t4 + 8, + 9), in units
              const uint32_t d = __shfl_sync(0xffffffffu, mt[kt][j], 8 * g + t4);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                uint32_t &h = bh[nt][kt][j], &lo = bl[nt][kt][j];
                const uint32_t p = ph[nt][kt][j], rest = pl[nt][kt][j];
                // p d = hi + lo: hi the rounded product, lo its exact rest and p_lo d
                if (!LO) {
                  h = hmul2(p, d);
                } else if (DUP) {  // hi in lanes with pn = pl = 0, lo in the others
                  h = hfma2(rest, d, hfma2(p, d, hmul2(pn[nt][kt][j], d)));
                } else {
                  h = hmul2(p, d);
                  lo = hfma2(rest, d, hfma2(p, d, h ^ 0x80008000u));
                }
              }
            }
          uint32_t va[2][4], vb[2][4];
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) {
            spread_codes<LO>(w[kt][2 * gi], va[kt]);
            spread_codes<LO>(w[kt][2 * gi + 1], vb[kt]);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float sum[4];
              mma_f16_zero(sum, va[0][2 * i], va[0][2 * i + 1], vb[0][2 * i], vb[0][2 * i + 1],
                           bh[nt][0][0], bh[nt][0][1]);
              mma_f16_16816(sum, va[1][2 * i], va[1][2 * i + 1], vb[1][2 * i], vb[1][2 * i + 1],
                            bh[nt][1][0], bh[nt][1][1]);
              if (LO && !DUP)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
                  mma_f16_16816(sum, va[kt][2 * i], va[kt][2 * i + 1], vb[kt][2 * i],
                                vb[kt][2 * i + 1], bl[nt][kt][0], bl[nt][kt][1]);
              add4(o[nt][g][i], sum);
            }
        }
      }
    };
    for (; blk < end_blk; ++blk) {
      // after a wait that ran out (status is set) the rest is only walked through
      if (ok) ok = mbar_wait_bounded(bar0 + 8 * stage, phase, a.status);
      if (blk >= mask_from)
        block(std::true_type());
      else
        block(std::false_type());
      __syncwarp();  // every lane is done with the stage
      if (to_copy > 0) copy(stage);
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }
    }

    // the item or the stretch ends: the item's output, or a piece of it
    {
      Item cur = s_cur[warp];
      const bool item_ends = blk == cur.nb;
      const int item = x - blk;  // the item's first block on the line
      const bool whole = item_ends && first_blk == 0;
      const int slot = 2 * warp + (x == w1 ? 1 : 0);
      float *piece = x == w1 ? reinterpret_cast<float *>(smem + warp * STAGES * kStage)
                             : heads + warp * kPiece;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int count = cur.count;
        l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], 1);
        l[nt] += __shfl_xor_sync(0xffffffffu, l[nt], 2);
        const float inv = whole ? (l[nt] > 0.f ? 1.f / l[nt] : (l[nt] == 0.f ? 0.f : NAN)) : 1.f;
        const float i0 = __shfl_sync(0xffffffffu, inv, 8 * t4), i1 = __shfl_sync(0xffffffffu, inv, 8 * t4 + 4);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float m0 = __shfl_sync(0xffffffffu, om[nt][0], 4 * (2 * g + 1) + t4),
                m1 = __shfl_sync(0xffffffffu, om[nt][1], 4 * (2 * g + 1) + t4);
          if (kSplit) {
            m0 += __shfl_xor_sync(0xffffffffu, m0, 2);
            m1 += __shfl_xor_sync(0xffffffffu, m1, 2);
          }
          const float in_units = power_of_two(__shfl_sync(0xffffffffu, unit_exponent(unit), 8 * g));
          float v[2][4];  // columns 2 t4 and 2 t4 + 1, dimensions 32 g + 4 r ..
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              float w = o[nt][g][i][c];
              if (kSplit) w += __shfl_xor_sync(0xffffffffu, w, 2);  // hi + lo
              v[c & 1][2 * i + (c >> 1)] = fmaf(w, code_unit<LO>(c >> 1) * in_units, (c & 1) ? m1 : m0);
            }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int col = nt * 8 + 2 * t4 + c;
            if (DUP && col >= 4) continue;
            if (whole) {
              if (col >= count * a.group) continue;
              const int tok = col / a.group;
              OutT *dst = reinterpret_cast<OutT *>(a.out) +
                          (((size_t)cur.b * a.tokens + tok) * a.n_heads + cur.h * a.group +
                           (col - tok * a.group)) * kD + 32 * g + 4 * r;
              const float f = c ? i1 : i0;
              OutT e[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) e[i] = from_float<OutT>(v[c][i] * f);
              *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(e);
            } else {
              float *dst = piece + col * kPieceRow + 32 * g + 4 * r;
#pragma unroll
              for (int i = 0; i < 4; i += 2)
                *reinterpret_cast<float2 *>(dst + i) = make_float2(v[c][i], v[c][i + 1]);
            }
          }
        }
        if (!whole && t4 == 0 && (!DUP || r < 4)) {
          piece[(nt * 8 + r) * kPieceRow + kD] = fmaf(mx[nt], cs[nt], -kBias);
          piece[(nt * 8 + r) * kPieceRow + kD + 1] = l[nt];
        }
      }
      if (!whole && lane == 0) {
        s_item[slot] = item;
        s_of[slot] = cur;
      }
      if (item_ends && x < w1) {
        next_item(cur);
        keep(s_cur[warp], cur);
        blk = 0;
      }
    }
  }
  if (!ok) {  // let this warp's last copies land before its shared memory goes
    for (int i = 0; i < min(STAGES, w1 - w0); ++i)
      mbar_wait_bounded(bar0 + 8 * i, (uint32_t)((w1 - w0 - 1 - i) / STAGES) & 1, a.status);
  }
  __syncthreads();

  // Join the pieces.  A slot per lane; an item's pieces are one per warp of a
  // range of warps: in the ring where the warp's stretch ended inside the item, its
  // head piece where the item ended first.  A warp takes a column of an item, a lane
  // four dimensions and one piece's statistics.
  const int my_item = lane < 2 * W ? s_item[lane] : -1;
  int task = 0, open0 = -1, open1 = -1;  // slots of items that go beyond this CTA
  for (uint32_t left = __ballot_sync(0xffffffffu, my_item >= 0); left;) {
    const int s0 = __ffs(left) - 1;
    const int item = __shfl_sync(0xffffffffu, my_item, s0);
    const uint32_t group = __ballot_sync(0xffffffffu, my_item == item) & left;
    left &= ~group;
    const int s1 = 31 - __clz(group);
    const int first_warp = s0 >> 1, n = (s1 >> 1) - first_warp + 1;
    const bool complete = item >= cta0 && item + s_of[s0].nb <= cta1;
    for (int col = 0; col < kCols; ++col, ++task) {
      if (task % W != warp) continue;
      auto piece_of = [&](int i) -> const float * {  // of warp first_warp + i
        return (i == n - 1 && !(s1 & 1)
                    ? heads + (first_warp + i) * kPiece
                    : reinterpret_cast<const float *>(smem + (first_warp + i) * STAGES * kStage)) +
               col * kPieceRow;
      };
      const float *ps = piece_of(min(lane, n - 1)) + kD;
      const float m = lane < n ? ps[0] : -INFINITY;
      const float top = warp_max(m);
      const float f = m == top ? 1.f : ex2(m - top);
      const float sum = warp_sum(lane < n ? f * ps[1] : 0.f);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int k = 0; k < n; ++k) {
        const float fk = __shfl_sync(0xffffffffu, f, k);
        const float4 w = *reinterpret_cast<const float4 *>(piece_of(k) + 4 * lane);
        v.x = fmaf(fk, w.x, v.x);
        v.y = fmaf(fk, w.y, v.y);
        v.z = fmaf(fk, w.z, v.z);
        v.w = fmaf(fk, w.w, v.w);
      }
      if (complete) {
        const Item of = s_of[s0];
        if (col >= of.count * a.group) continue;
        const int tok = a.tokens == 1 ? 0 : col / a.group;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        OutT e[4] = {from_float<OutT>(v.x * inv), from_float<OutT>(v.y * inv),
                     from_float<OutT>(v.z * inv), from_float<OutT>(v.w * inv)};
        *reinterpret_cast<uint2 *>(reinterpret_cast<OutT *>(a.out) +
                                   (((size_t)of.b * a.tokens + tok) * a.n_heads + of.h * a.group +
                                    (col - tok * a.group)) * kD + 4 * lane) =
            *reinterpret_cast<const uint2 *>(e);
      } else {  // at most one item that began before this CTA's stretch, one that goes on
        float *mine = a.parts + (((size_t)blockIdx.x * 2 + (item < cta0 ? 0 : 1)) * kMaxCols + col) *
                                    kPieceRow;
        *reinterpret_cast<float4 *>(mine + 4 * lane) = v;
        if (lane == 0) *reinterpret_cast<float2 *>(mine + kD) = make_float2(top, sum);
      }
    }
    if (!complete) (item < cta0 ? open0 : open1) = s0;
  }
  if (open0 < 0 && open1 < 0) return;
  // the last CTA of such an item to arrive joins the CTAs' parts
  __threadfence();
  __syncthreads();
  if (threadIdx.x < 2) {
    const int s = threadIdx.x ? open1 : open0;
    bool last = false;
    if (s >= 0) {
      const int item = s_item[s], c0 = item / quota;
      last = atomicAdd(a.arrivals + c0, 1) == (item + s_of[s].nb - 1) / quota - c0;
      if (last) a.arrivals[c0] = 0;
    }
    s_last[threadIdx.x] = last;
  }
  __syncthreads();
  __threadfence();
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    if (!s_last[i]) continue;
    const int s = i ? open1 : open0, item = s_item[s];
    const Item of = s_of[s];
    join_parts<NT == 1 ? 2 : 4, OutT>(a, of, item / quota, (item + of.nb - 1) / quota, warp, W);
  }
}

// warps (as many on each SM quarter: 14 of them left two quarters idle for a sixth of
// the time) and ring stages per column count: 160-184 KB in flight per SM
template <int NT, bool DUP>
struct FewShape {
  static constexpr int warps = NT == 1 ? 16 : 8;
  static constexpr int stages = NT == 1 ? 2 : 4;
  static constexpr size_t smem(int batch) {
    return (size_t)warps * stages * kStage + sizeof(int) * (batch + 1);
  }
};
// the CTAs' parts, then the warps' head pieces
constexpr size_t few_scratch_floats(int sm_count) {
  return ((size_t)2 * kMaxCols + 16 * kMaxCols) * sm_count * kPieceRow;
}

template <int NT, bool DUP, class OutT>
constexpr auto few_kernel() {
  using S = FewShape<NT, DUP>;
  return kv4_attn_few_kernel<NT, DUP, S::warps, S::stages, OutT>;
}

template <int NT, bool DUP, class OutT>
int few_launch(mlm_ctx *ctx, const Kv4AttnArgs &a) {
  using S = FewShape<NT, DUP>;
  return check_launch_pdl(ctx,
                          launch_pdl(few_kernel<NT, DUP, OutT>(), dim3(ctx->sm_count),
                                     dim3(S::warps * 32), S::smem(a.batch), ctx->stream, a),
                          "mlm_attn_kv4");
}
template <class OutT>
int few(mlm_ctx *ctx, const Kv4AttnArgs &a) {
  const int cols = a.tokens * a.group;
  if (cols <= 4) return few_launch<1, true, OutT>(ctx, a);
  if (cols <= 8) return few_launch<1, false, OutT>(ctx, a);
  return few_launch<2, false, OutT>(ctx, a);
}

template <int NT, bool DUP, class OutT>
int few_init(mlm_ctx *ctx) {
  MLM_CUDA_TRY(ctx, cudaFuncSetAttribute(few_kernel<NT, DUP, OutT>(),
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)FewShape<NT, DUP>::smem(MLM_KV4_MAX_BATCH)));
  return MLM_OK;
}

}  // namespace

int kv4_attn_init(mlm_ctx *ctx) {
  int st = few_init<1, true, __half>(ctx);
  if (st == MLM_OK) st = few_init<1, false, __half>(ctx);
  if (st == MLM_OK) st = few_init<2, false, __half>(ctx);
  if (st == MLM_OK) st = few_init<1, true, __nv_bfloat16>(ctx);
  if (st == MLM_OK) st = few_init<1, false, __nv_bfloat16>(ctx);
  if (st == MLM_OK) st = few_init<2, false, __nv_bfloat16>(ctx);
  if (st == MLM_OK) st = kv4_attn_many_init(ctx);
  if (st != MLM_OK) return st;
  const size_t parts = std::max(sizeof(float) * few_scratch_floats(ctx->sm_count),
                                kv4_many_parts_bytes(ctx->sm_count));
  if (cudaMalloc(&ctx->kv4_parts, parts) != cudaSuccess ||
      cudaMalloc(&ctx->kv4_arrivals, sizeof(int) * (ctx->sm_count + 1 + kKv4PlanInts)) != cudaSuccess)
    return set_error(ctx, MLM_ERR_ALLOC, "mlm_attn_kv4: scratch");
  MLM_CUDA_TRY(ctx, cudaMemset(ctx->kv4_arrivals, 0, sizeof(int) * ctx->sm_count));
  return MLM_OK;
}

int kv4_attn_few(mlm_ctx *ctx, const Kv4AttnArgs &a, int out_type) {
  return out_type == MLM_TYPE_F16 ? few<__half>(ctx, a) : few<__nv_bfloat16>(ctx, a);
}

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
  const int group = n_heads / cache->n_kv_heads;
  Kv4AttnArgs a;
  a.kc = reinterpret_cast<const uint8_t *>(cache->k);
  a.vc = reinterpret_cast<const uint8_t *>(cache->v);
  a.q = reinterpret_cast<const __half *>(q);
  a.out = out;
  a.lens = lens;
  a.counts = counts;
  a.parts = ctx->kv4_parts;
  a.arrivals = ctx->kv4_arrivals;
  a.plan = ctx->kv4_arrivals + (ctx->sm_count + 1) / 2 * 2;
  a.status = ctx->dev_status;
  a.batch = cache->batch;
  a.tokens = tokens;
  a.n_heads = n_heads;
  a.n_kv = cache->n_kv_heads;
  a.group = group;
  a.capacity = cache->capacity;
  return (long long)tokens * group <= kMaxCols ? kv4_attn_few(ctx, a, out_type)
                                               : kv4_attn_many(ctx, a, out_type);
}
