// kv4_attn_many.cu -- attention over the 4-bit KV cache for many rows: prompt
// chunks, and more than 16 (token, head) pairs per KV head in general.
//
// The rows of one (sequence, KV head) are its (token, query head of the group)
// pairs, token first, so a group's heads share every key tile.  A CTA takes 256
// rows (two tiles of 128) against tiles of 128 keys, both products on tcgen05
// with fp32 accumulators in TMEM (M = N = 128):
//   - 4 warps each turn a key tile's cache rows into fp16 K and V in shared memory
//     (a thread per key; one rounding of m + d c, as the read-back gives it), two
//     buffers of each, handed back as soon as their last product is done;
//   - one thread issues S = Q K^T and O += P V, the two row tiles in turn, so
//     that one tile's softmax runs while the other's products do;
//   - 4 warps per row tile do the softmax, a thread per row: S from TMEM, the
//     weights back as fp16 over it, where the second product reads them as its A
//     operand.
// The running maximum follows only when a score leads it by more than 2^8, so the
// accumulator in TMEM is rescaled once or twice in a row's life, as a rule.  The weights
// are 2^(s - max + 7): at most 2^15, and held to 2^-32 of the largest, as the many small
// ones of a long cache want (2^17 of them are off by 2^-15 together).  Scores, maxima and
// sums are fp32.  For a bf16 output K, V and the weights are fp16 operands, each rounded
// once; an fp16 output, eight times finer, would show that (up to three times its own
// rounding), so there each is hi + lo: two products for the scores, three for O.
//
// A product's accumulators are cut off, not rounded, by up to 2^-23 each time, and 131072
// keys in one accumulator shrank by 4e-4.  So after 128 key tiles (512 for a bf16 output)
// O is added to the part of the scratch that the item would leave, and the next products
// start from zero.  All CTAs at once move 38 MB each way in such a fold, some 10 us: every
// 64 tiles 1024 tokens at 32768 keys to bf16 took 558 us, 520 as it is.
//
// V^T is the N-major B operand of the second product: both K and V lie in
// shared memory as [key][dimension] in the 128-byte swizzle, the eight
// elements of a code word in the order its masks give (0 4 1 5 2 6 3 7); Q is
// stored in the same order and the output columns are put back.
//
// The tiles of all (sequence, 256 rows, KV head) items form one line that is cut
// into equal stretches, one per CTA, from the lengths in device memory.  An item
// that several CTAs share leaves fp32 parts in the context's scratch, which a
// second kernel joins in order.
//
// Measured: 1024 tokens at 8192, 32/8 heads, 147 us, 877 TFLOP/s (162 us at the card's
// power limit, 1810 MHz for 1965), the tensor pipe 44 % active: bound by the chain S,
// softmax, P, P V of the two row tiles (144 us without exponentials, maxima and
// dequantization, 107 us without the products).  At 96 registers a thread at launch the
// kernel spills 350 bytes a thread (480 for fp16 outputs).  Half tiles with a thread per
// row tile issuing took 167 us, handing P over in halves 170, the maximum in a pass
// before the exponentials 164.  To fp16: 338 us.
//
// A NaN in a cache row reaches every token that sees the row and no other: a
// masked weight is 0, but 0 x NaN is not, so a value row with NaN scales goes in
// as zeros and makes its key NaN instead.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "kv4_common.cuh"
#include "q4k_gemv_common.cuh"

namespace mlm {
namespace {

constexpr int kTile = 128;          // rows of a row tile, keys of a key tile
constexpr int kRows = 2 * kTile;    // rows of an item
constexpr int kSoftWarps = 8, kDqWarps = 8;  // the latter: 4 for K, 4 for V
constexpr int kMmaWarp = kSoftWarps + kDqWarps;
constexpr int kThreads = 32 * (kMmaWarp + 4);  // whole warpgroups; three warps idle
// registers per thread: at launch, then per role; the roles' sum stays below the
// launch's (65536 / kThreads rounded down to a multiple of 8)
constexpr int kLaunchRegs = 96, kSoftRegs = 136, kDqRegs = 72, kMmaRegs = 64;
static_assert(32 * kSoftWarps * kSoftRegs + 32 * kDqWarps * kDqRegs + 128 * kMmaRegs <=
                  kThreads * kLaunchRegs,
              "the roles' registers");
constexpr int kSub = kTile * 128;           // 64 dimensions of a tile: 128 rows x 128 bytes
constexpr int kOperand = 2 * kSub;          // 32 KB: Q, K or V of a tile
constexpr int kOffKv = 2 * kOperand;        // after Q of two tiles
constexpr int kOffBar = kOffKv + 4 * kOperand;
enum { kQfull = 0, kSfull = 1, kPfull = 3, kOfull = 5, kKfull = 7, kVfull = 9, kKempty = 11, kVempty = 13,
       kDrain = 15, kBars = 16 };
constexpr int kOffTmem = kOffBar + 8 * kBars;
constexpr int kOffLine = kOffTmem + 16;     // [batch + 1] 64-bit offsets
constexpr size_t smem_bytes(int batch) { return kOffLine + 8 * (size_t)(batch + 1); }
constexpr int kTmemCols = 512;  // S/P of tile 0 and 1, O of tile 0 and 1
constexpr int kPartFloats = kRows * (kKv4D + 2);  // o, then m and l
constexpr float kScale2 = kInvSqrtD * kLog2e;
constexpr float kBias = 7.f, kLead = 8.f / kScale2;
// key tiles whose products O sums in TMEM: 24 products a tile for an fp16 output, 8 for bf16
constexpr int fold_of(bool exact) { return exact ? 128 : 512; }

// instruction descriptors: fp16 A and B, fp32 accumulators, M = N = 128; B K-major
// (S = Q K^T) or N-major (O = P V)
constexpr uint32_t kIdescS = (1u << 4) | ((kTile >> 3) << 17) | ((kTile >> 4) << 24);
constexpr uint32_t kIdescO = kIdescS | (1u << 16);

// Matrix descriptors of the 128-byte swizzle: rows of 128 bytes in 8-row atoms
// of 1024 bytes, 16-byte chunk c of row r at c ^ (r & 7); version 1, layout type
// 2.  K-major: atoms 1024 bytes apart along the rows.  N-major: 8-key groups
// 1024 bytes apart, 64-dimension halves kSub bytes apart.
// The high words are alike; a low word is the address in 16-byte units (shared
// memory's addresses fit the field) and the other stride, so a step along K is one
// addition.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k_major(uint32_t addr) { return (addr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_n_major(uint32_t addr) {
  return (addr >> 4) | ((uint32_t)(kSub >> 4) << 16);
}
// byte offset of 16-byte chunk c (0 .. 15) of row r in an operand
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (uint32_t)((c >> 3) * kSub + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// One thread issues all products, and each takes the tensor cores 64 cycles: the
// operands' descriptors are low words that change by constants.
template <bool ACC>
__device__ __forceinline__ void mma_smem(uint32_t d, uint32_t a, uint32_t b) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %5, 0;\n"
      " mov.b64 da, {%1, %3};\n mov.b64 db, {%2, %3};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n}" ::"r"(d),
      "r"(a), "r"(b), "n"(kDescHi), "n"(kIdescS), "n"(ACC ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %5, 0;\n"
      " mov.b64 db, {%2, %3};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n}" ::"r"(d),
      "r"(a), "r"(b), "n"(kDescHi), "n"(kIdescO), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   bar)
               : "memory");
}
__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// 32 columns of the warp's lanes; the values are there after tmem_wait_ld, which
// names them so that no use moves above it
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
        "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
        "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]),
                 "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]),
                 "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]),
                 "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
                 "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29])
               :
               : "memory");
  asm volatile("" : "+r"(v[30]), "+r"(v[31])::"memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t *v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
      "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]),
      "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]),
      "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// packed fp32 pairs
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// x and y as fp16 pairs hi + lo
__device__ __forceinline__ void split_f16(float x, float y, uint32_t &hi, uint32_t &lo) {
  hi = pack_f16(x, y);
  const float2 h = unpack_f16(hi);
  lo = pack_f16(x - h.x, y - h.y);
}

__device__ __forceinline__ int row_tiles(int count, int group) {
  return (count * group + kRows - 1) / kRows;
}
// key tiles of a sequence's rt-th 256 rows: up to what their last token sees
__device__ __forceinline__ int key_tiles(int len, int count, int group, int rt) {
  const int last = min(count - 1, ((rt + 1) * kRows - 1) / group);
  return max(0, (len - count + last + 1 + kTile - 1) / kTile);
}

// Key tiles kt0 .. kt1 of nkt of an item: a CTA's stretch is a sequence of these,
// which every role walks alike.
struct Part {
  int b, rt, h, kt0, kt1, nkt, len, count;
};
struct Walk {
  const Kv4AttnArgs &a;
  const long long *off;  // the line's offsets per sequence
  long long x, x1;
  Part p;
  __device__ Walk(const Kv4AttnArgs &a_, const long long *off_, long long x0, long long x1_)
      : a(a_), off(off_), x(x0), x1(x1_), p{} {
    if (x >= x1) return;
    int lo = 0, hi = a.batch;  // the last sequence with off <= x
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (off[mid] <= x) lo = mid; else hi = mid;
    }
    p.b = lo;
    seq_shape(a, lo, p.len, p.count);
    long long y = x - off[lo];
    for (;; ++p.rt) {
      p.nkt = key_tiles(p.len, p.count, a.group, p.rt);
      const long long span = (long long)p.nkt * a.n_kv;
      if (y < span) break;
      y -= span;
    }
    p.h = (int)(y / p.nkt);
    p.kt1 = (int)(y - (long long)p.h * p.nkt);  // where the first part begins
    --p.h;  // next() moves on from the item before
    first = true;
  }
  bool first = false;
  __device__ bool next() {
    if (x >= x1) return false;
    const int begin = first ? p.kt1 : 0;
    first = false;
    if (++p.h == a.n_kv) {
      p.h = 0;
      do {
        ++p.rt;
        while (p.rt >= row_tiles(p.count, a.group) || off[p.b + 1] == off[p.b]) {
          ++p.b;
          p.rt = 0;
          seq_shape(a, p.b, p.len, p.count);
        }
        p.nkt = key_tiles(p.len, p.count, a.group, p.rt);
      } while (p.nkt == 0);
    }
    p.kt0 = begin;
    p.kt1 = (int)min((long long)p.nkt, begin + (x1 - x));
    x += p.kt1 - p.kt0;
    return true;
  }
};

// one word of codes to eight fp16 values in the order 0 4 1 5 2 6 3 7, and with LO
// what rounding left of them, as fp16
template <bool LO>
__device__ __forceinline__ void values8(uint32_t w, __half2 d, __half2 m, uint4 &value, uint4 &rest) {
  // codes in the mantissa of 1024 (of 64 where they sit 4 bits higher)
  const __half2 one = __float2half2_rn(-1024.f), low = __float2half2_rn(-64.f),
                sixteenth = __float2half2_rn(0.0625f);
  const uint64_t df = pair(__low2float(d), __low2float(d)), mf = pair(__low2float(m), __low2float(m));
  uint32_t v[4], e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = i < 2 ? w : w >> 8;
    const uint32_t a = (x & (i & 1 ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
    const __half2 ha = *reinterpret_cast<const __half2 *>(&a);
    const __half2 c = i & 1 ? __hfma2(ha, sixteenth, low) : __hadd2(ha, one);
    const __half2 h = __hfma2(c, d, m);
    v[i] = *reinterpret_cast<const uint32_t *>(&h);
    if (LO) {
      const float2 cf = __half22float2(c), hf = __half22float2(h);
      const float2 r = unpair(add2(fma2(pair(cf.x, cf.y), df, mf), pair(-hf.x, -hf.y)));
      e[i] = pack_f16(r.x, r.y);
    }
  }
  value = make_uint4(v[0], v[1], v[2], v[3]);
  if (LO) rest = make_uint4(e[0], e[1], e[2], e[3]);
}
template <class OutT>
__global__ void __launch_bounds__(kThreads, 1) kv4_attn_many_kernel(Kv4AttnArgs a) {
  // hi + lo operands, each in one buffer of the two instead of one in two
  constexpr bool EXACT = std::is_same<OutT, __half>::value;
  constexpr uint32_t kStages = EXACT ? 1 : 2;
  constexpr int kFold = fold_of(EXACT);
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = (uint32_t)__cvta_generic_to_shared(smem);
  const uint32_t bar = sbase + kOffBar;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + kOffTmem);
  long long *s_off = reinterpret_cast<long long *>(smem + kOffLine);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(bar + 8 * kQfull, 32 * kSoftWarps);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar + 8 * (kSfull + i), 1);
      mbar_init(bar + 8 * (kPfull + i), kTile);
      mbar_init(bar + 8 * (kOfull + i), 1);
      mbar_init(bar + 8 * (kKfull + i), kDqWarps / 2);
      mbar_init(bar + 8 * (kVfull + i), kDqWarps / 2);
      mbar_init(bar + 8 * (kKempty + i), 1);
      mbar_init(bar + 8 * (kVempty + i), 1);
    }
    mbar_init(bar + 8 * kDrain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     (uint32_t)__cvta_generic_to_shared(tmem_slot)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pdl_wait_then_release();

  // the line: key tiles per sequence, then their running sum
  for (int b = warp; b < a.batch; b += kThreads / 32) {
    int len, count;
    seq_shape(a, b, len, count);
    long long n = 0;
    for (int rt = lane; rt < row_tiles(count, a.group); rt += 32)
      n += (long long)key_tiles(len, count, a.group, rt) * a.n_kv;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if (lane == 0) {
      s_off[b + 1] = n;
      if (blockIdx.x == 0 && seq_outside(a, b)) report_outside(a.status);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0) {
    long long run = 0;
    s_off[0] = 0;
    for (int b = 1; b <= a.batch; ++b) s_off[b] = run += s_off[b];
  }
  __syncthreads();
  const uint32_t tmem = *tmem_slot;
  const long long total = s_off[a.batch];
  const long long quota = max(1ll, (total + gridDim.x - 1) / gridDim.x);
  const long long x0 = min(total, blockIdx.x * quota), x1 = min(total, x0 + quota);
  if (blockIdx.x == 0) {  // the cut, for the joining kernel
    long long *plan = reinterpret_cast<long long *>(a.plan);
    if (threadIdx.x == 0) plan[0] = quota;
    for (int b = threadIdx.x; b <= a.batch; b += kThreads) plan[1 + b] = s_off[b];
  }
  // tokens that attend to nothing: the first count - len of a sequence
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    int len, count;
    seq_shape(a, b, len, count);
    OutT *o = reinterpret_cast<OutT *>(a.out) + (size_t)b * a.tokens * a.n_heads * kKv4D;
    const long long n = (long long)max(0, count - len) * a.n_heads * kKv4D;
    for (long long i = threadIdx.x; i < n; i += kThreads) o[i] = from_float<OutT>(0.f);
  }

  Walk walk(a, s_off, x0, x1);
  bool ok = true;
  if (warp < kSoftWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    // ---- softmax: a thread per row of tile `tile` --------------------------------
    const int tile = warp >> 2, r = threadIdx.x & (kTile - 1);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + tile * kTile, to = tmem + lanes + (2 + tile) * kTile;
    uint32_t n_s = 0, n_q = 0, n_item = 0;
    while (ok && walk.next()) {
      const Part p = walk.p;
      const int live = p.count * a.group - p.rt * kRows;  // rows of the item
      const int row = p.rt * kRows + tile * kTile + r;
      const bool mine = tile * kTile + r < live;
      const int tok = mine ? row / a.group : 0;
      // (a row past the item sees all of its zero scores: the mask for its sake cost 64 rows
      // x 16 sequences of 16000 296 us, 238 without)
      const int seen = mine ? max(0, p.len - p.count + tok + 1) : INT_MAX;
      const size_t at = (((size_t)p.b * a.tokens + tok) * a.n_heads + p.h * a.group +
                         (row - tok * a.group)) * kKv4D;
      // Q in the order of the codes: half a warp per row
      uint8_t *s_q = smem + tile * kOperand;
      auto row_at = [&](int i) {  // where row i of the warp's 32 lies in q and out
        return ((uint64_t)__shfl_sync(0xffffffffu, (uint32_t)(at >> 32), i) << 32) |
               __shfl_sync(0xffffffffu, (uint32_t)at, i);
      };
      const uint32_t rows = __ballot_sync(0xffffffffu, mine);
      const int r0 = (warp & 3) * 32;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int j = 2 * i + (lane >> 4), c = lane & 15;
        const uint64_t from = row_at(j);
        uint4 v = make_uint4(0, 0, 0, 0);
        if ((rows >> j) & 1) v = *reinterpret_cast<const uint4 *>(a.q + from + 8 * c);
        *reinterpret_cast<uint4 *>(s_q + chunk_at(r0 + j, c)) =
            make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                       __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc_fence_before();
      arrive(bar + 8 * kQfull);
      if (tile * kTile >= live) {  // no row of this tile: its products do not run
        // not past the other tile: its arrivals for this item come first
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar + 8 * kQfull, n_q++ & 1, a.status));
        continue;
      }
      ++n_q;
      // the CTA's part of the item: [4 columns][row], then the rows' maxima and sums.  An
      // item without parts folds into the second, which only the stretch's last item may
      // leave.  (Found anew where it is used: the loop has no registers to spare.)
      auto part_at = [&] {
        const long long item = walk.x - p.kt1;  // the item's first tile on the line
        return a.parts + ((size_t)blockIdx.x * 2 + (item < x0 ? 0 : 1)) * kPartFloats + 4 * (tile * kTile + r);
      };
      auto fold = [&](bool more, float m) {
        float4 *part_o = reinterpret_cast<float4 *>(part_at());
        float *part_m = reinterpret_cast<float *>(part_o) + kRows * kKv4D - 3 * (tile * kTile + r);
        const float was = more ? *part_m : m;
        const float f = was == m ? 1.f : ex2((was - m) * kScale2);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(to + 32 * c, o);
          tmem_wait_ld(o);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float4 *dst = part_o + (8 * c + j) * kRows;
            const float4 x = more ? *dst : make_float4(0.f, 0.f, 0.f, 0.f);
            *dst = make_float4(fmaf(f, x.x, __uint_as_float(o[4 * j])),
                               fmaf(f, x.y, __uint_as_float(o[4 * j + 1])),
                               fmaf(f, x.z, __uint_as_float(o[4 * j + 2])),
                               fmaf(f, x.w, __uint_as_float(o[4 * j + 3])));
          }
        }
        *part_m = m;
      };
      float m = -INFINITY;
      uint64_t l2 = 0;
      for (int first = p.kt0; first < p.kt1; first += kFold) {
        const int last = min(p.kt1, first + kFold);
        if (first > p.kt0) {
          // The sums of the last kFold tiles, in the order of the products, are added to
          // those before; once the next S is there they are complete
          ok = __all_sync(0xffffffffu,
                          mbar_wait_bounded(bar + 8 * (kSfull + tile), n_s & 1, a.status));
          if (!ok) break;
          tc_fence_after();
          fold(first - p.kt0 > kFold, m);
        }
        for (int kt = first; kt < last; ++kt) {
          ok = __all_sync(0xffffffffu,
                          mbar_wait_bounded(bar + 8 * (kSfull + tile), n_s & 1, a.status));
          if (!ok) break;
          ++n_s;
          tc_fence_after();
          const int lim = seen - kt * kTile;  // keys of the tile that the row sees
          auto weights = [&](auto mask_tag) {
            constexpr bool MASK = decltype(mask_tag)::value;
            uint32_t s[2][32];
            float m2 = m == -INFINITY ? 0.f : fmaf(-m, kScale2, kBias);
            tmem_ld32(ts, s[0]);
  #pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t(&v)[32] = s[c & 1];
              tmem_wait_ld(v);
              if (c < 3) tmem_ld32(ts + 32 * (c + 1), s[(c + 1) & 1]);
              float top = -INFINITY, top1 = -INFINITY;
  #pragma unroll
              for (int k = 0; k < 32; k += 2) {
                if (MASK) {
                  if (32 * c + k >= lim) v[k] = 0xFF800000u;
                  if (32 * c + k + 1 >= lim) v[k + 1] = 0xFF800000u;
                }
                top = fmaxf(top, __uint_as_float(v[k]));
                top1 = fmaxf(top1, __uint_as_float(v[k + 1]));
              }
              top = fmaxf(top, top1);
              if (__any_sync(0xffffffffu, top > m + kLead)) {
                // a new maximum: what has been summed against the old one is scaled,
                // O, l and this tile's weights so far
                if (c < 3) tmem_wait_ld(s[(c + 1) & 1]);
                const float up = fmaxf(m, top);
                const float f = up == m ? 1.f : ex2((m - up) * kScale2);
                if (kt > first) {
  #pragma unroll 1
                  for (int j = 0; j < 4; ++j) {
                    uint32_t o[32];
                    tmem_ld32(to + 32 * j, o);
                    tmem_wait_ld(o);
  #pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                    tmem_st32(to + 32 * j, o);
                  }
                }
                tmem_wait_st();
                if (EXACT) {
  #pragma unroll 1
                  for (int j = 0; j < c; ++j) {
                    uint32_t o[32];
                    tmem_ld32(ts + 32 * j, o);
                    tmem_wait_ld(o);
  #pragma unroll
                    for (int k = 0; k < 16; ++k) {
                      const float2 h = unpack_f16(o[k]), e = unpack_f16(o[16 + k]);
                      split_f16((h.x + e.x) * f, (h.y + e.y) * f, o[k], o[16 + k]);
                    }
                    tmem_st32(ts + 32 * j, o);
                  }
                } else {
  #pragma unroll 1
                  for (int j = 0; j < (c + 1) / 2; ++j) {  // 64 weights at a time
                    uint32_t o[32];
                    tmem_ld32(ts + 32 * j, o);
                    tmem_wait_ld(o);
                    uint32_t h[16];
  #pragma unroll
                    for (int half = 0; half < 2; ++half) {
  #pragma unroll
                      for (int k = 0; k < 16; ++k) {
                        const float2 e = unpack_f16(o[16 * half + k]);
                        h[k] = pack_f16(e.x * f, e.y * f);
                      }
                      if (2 * j + half < c) tmem_st16(ts + 32 * j + 16 * half, h);
                    }
                  }
                }
                tmem_wait_st();
                const float2 l = unpair(l2);
                l2 = pair(l.x * f, l.y * f);
                m = up;
                m2 = m == -INFINITY ? 0.f : fmaf(-m, kScale2, kBias);
              }
              const uint64_t mm = pair(m2, m2), cc = pair(kScale2, kScale2);
              uint32_t w[16], rest[16];
              // (a chunk's sum first: 2^16 equal weights added one by one would be rounded the
              // same way each, by up to 2^-9 of a weight)
              uint64_t sum2 = 0;
  #pragma unroll
              for (int k = 0; k < 32; k += 2) {
                const float2 e =
                    unpair(fma2(pair(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), cc, mm));
                const float p0 = ex2(e.x), p1 = ex2(e.y);
                sum2 = k == 0 ? pair(p0, p1) : add2(sum2, pair(p0, p1));
                if (EXACT)
                  split_f16(p0, p1, w[k / 2], rest[k / 2]);
                else
                  w[k / 2] = pack_f16(p0, p1);
              }
              l2 = add2(l2, sum2);
              // over scores that have been read
              tmem_st16(ts + (EXACT ? 32 : 16) * c, w);
              if (EXACT) tmem_st16(ts + 32 * c + 16, rest);
            }
          };
          if (__any_sync(0xffffffffu, lim < kTile))
            weights(std::true_type());
          else
            weights(std::false_type());
          tmem_wait_st();
          tc_fence_before();
          arrive(bar + 8 * (kPfull + tile));
        }
        if (!ok) break;
      }
      if (!ok) break;
      ok = __all_sync(0xffffffffu,
                      mbar_wait_bounded(bar + 8 * (kOfull + tile), n_item & 1, a.status));
      if (!ok) break;
      ++n_item;
      tc_fence_after();
      const float2 l = unpair(l2);
      const float sum = l.x + l.y;
      const bool whole = p.kt0 == 0 && p.kt1 == p.nkt;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      float4 *part_o = reinterpret_cast<float4 *>(part_at());
      float *part_m = reinterpret_cast<float *>(part_o) + kRows * kKv4D - 3 * (tile * kTile + r);
      const bool folded = p.kt1 - p.kt0 > kFold;
      const float was = folded ? *part_m : m;
      const float f_was = was == m ? 1.f : ex2((was - m) * kScale2);
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t o[32];
        tmem_ld32(to + 32 * c, o);
        tmem_wait_ld(o);
        if (folded) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 x = part_o[(8 * c + j) * kRows];
            o[4 * j] = __float_as_uint(fmaf(f_was, x.x, __uint_as_float(o[4 * j])));
            o[4 * j + 1] = __float_as_uint(fmaf(f_was, x.y, __uint_as_float(o[4 * j + 1])));
            o[4 * j + 2] = __float_as_uint(fmaf(f_was, x.z, __uint_as_float(o[4 * j + 2])));
            o[4 * j + 3] = __float_as_uint(fmaf(f_was, x.w, __uint_as_float(o[4 * j + 3])));
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float e[8];  // columns 0 4 1 5 2 6 3 7 back in order
#pragma unroll
          for (int k = 0; k < 8; ++k) e[(k >> 1) + 4 * (k & 1)] = __uint_as_float(o[8 * j + k]);
          if (whole) {  // by way of Q's place, which no product reads any more
            OutT h[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) h[k] = from_float<OutT>(e[k] * inv);
            *reinterpret_cast<uint4 *>(s_q + chunk_at(r, 4 * c + j)) =
                *reinterpret_cast<const uint4 *>(h);
          } else {
            float4 *dst = part_o + (8 * c + 2 * j) * kRows;
            dst[0] = make_float4(e[0], e[1], e[2], e[3]);
            dst[kRows] = make_float4(e[4], e[5], e[6], e[7]);
          }
        }
      }
      if (whole) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = 2 * i + (lane >> 4), c = lane & 15;
          const uint64_t to_row = row_at(j);
          if ((rows >> j) & 1)
            *reinterpret_cast<uint4 *>(reinterpret_cast<OutT *>(a.out) + to_row + 8 * c) =
                *reinterpret_cast<const uint4 *>(s_q + chunk_at(r0 + j, c));
        }
        __syncwarp();
      } else {
        part_m[0] = m * kScale2;
        part_m[kRows] = sum;
      }
    }
  } else if (warp < kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kDqRegs));
    // ---- cache rows to fp16 operands: a thread per key of the tile ----------------
    const int key = (threadIdx.x - 32 * kSoftWarps) & (kTile - 1);
    const bool is_v = warp >= kSoftWarps + kDqWarps / 2;
    const uint8_t *cache = is_v ? a.vc : a.kc;
    const uint32_t full = bar + 8 * (is_v ? kVfull : kKfull), empty = bar + 8 * (is_v ? kVempty : kKempty);
    uint32_t n_kv = 0;
    uint4 raw[5], v_scales = {};  // K's threads also look at their key's value scales
    auto load = [&](const Part &p, int kt) {
      const int j = kt * kTile + key;
      if (j < p.len) {
        const size_t at = (((size_t)p.b * a.n_kv + p.h) * a.capacity + j) * kKv4Row;
#pragma unroll
        for (int i = 0; i < 5; ++i) raw[i] = *reinterpret_cast<const uint4 *>(cache + at + 16 * i);
        v_scales = is_v ? raw[4] : *reinterpret_cast<const uint4 *>(a.vc + at + 64);
      } else {  // past the sequence: zeros
#pragma unroll
        for (int i = 0; i < 5; ++i) raw[i] = make_uint4(0, 0, 0, 0);
        v_scales = raw[4];
      }
    };
    bool more = walk.next();
    int kt = walk.p.kt0;
    if (more) load(walk.p, kt);
    while (more) {
      const uint32_t buf = n_kv % kStages;
      if (n_kv >= kStages) {
        ok = __all_sync(0xffffffffu,
                        mbar_wait_bounded(empty + 8 * buf, (n_kv / kStages - 1) & 1, a.status));
        if (!ok) break;
      }
      uint4 cur[5];
#pragma unroll
      for (int i = 0; i < 5; ++i) cur[i] = raw[i];
      if (not_finite(v_scales.x) || not_finite(v_scales.y) || not_finite(v_scales.z) ||
          not_finite(v_scales.w)) {
        const uint32_t x = is_v ? 0u : 0x7FFF7FFFu;
        cur[4] = make_uint4(x, x, x, x);
      }
      if (++kt == walk.p.kt1) {
        more = walk.next();
        kt = walk.p.kt0;
      }
      if (more) load(walk.p, kt);
      uint8_t *dst = smem + kOffKv + (2 * buf + is_v) * kOperand;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t dm = u4_get(cur[4], g);
        const uint32_t dd = __byte_perm(dm, dm, 0x1010), mm = __byte_perm(dm, dm, 0x3232);
        const __half2 d = *reinterpret_cast<const __half2 *>(&dd),
                      m = *reinterpret_cast<const __half2 *>(&mm);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint4 value, rest;
          values8<EXACT>(u4_get(cur[g], i), d, m, value, rest);
          *reinterpret_cast<uint4 *>(dst + chunk_at(key, 4 * g + i)) = value;
          if (EXACT) *reinterpret_cast<uint4 *>(dst + 2 * kOperand + chunk_at(key, 4 * g + i)) = rest;
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive(full + 8 * buf);
      ++n_kv;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMmaRegs));
    if (warp == kMmaWarp && lane == 0) {
    // ---- the products -----------------------------------------------------------
    uint32_t n_kv = 0, n_p[2] = {0, 0}, n_item = 0;
    const uint32_t q0 = desc_k_major(sbase), k0 = desc_k_major(sbase + kOffKv),
                   v0 = desc_n_major(sbase + kOffKv + kOperand);
    auto scores = [&](int tile, uint32_t buf) {
      const uint32_t q = q0 + tile * (kOperand >> 4), kb = k0 + buf * (2 * kOperand >> 4);
      const uint32_t d = tmem + tile * kTile;
      mma_smem<false>(d, q, kb);
#pragma unroll
      for (int k = 1; k < (EXACT ? 16 : 8); ++k) {
        constexpr int kStep = 32 >> 4, kHalf = kSub >> 4, kLo = 2 * kOperand >> 4;
        mma_smem<true>(d, q + ((k >> 2) & 1) * kHalf + (k & 3) * kStep,
                       kb + (k >> 3) * kLo + ((k >> 2) & 1) * kHalf + (k & 3) * kStep);
      }
      commit(bar + 8 * (kSfull + tile));
    };
    auto ready = [&](int which, uint32_t n) {
      const bool in_time = mbar_wait_bounded(bar + 8 * (which + n % kStages), (n / kStages) & 1, a.status);
      tc_fence_after();
      return in_time;
    };
    while (ok && walk.next()) {
      const Part p = walk.p;
      const int tiles = p.count * a.group - p.rt * kRows > kTile ? 2 : 1;
      ok = mbar_wait_bounded(bar + 8 * kQfull, n_item & 1, a.status) && ready(kKfull, n_kv);
      if (!ok) break;
      ++n_item;
      for (int i = 0; i < tiles; ++i) scores(i, n_kv % kStages);
      commit(bar + 8 * (kKempty + n_kv % kStages));
      for (int kt = p.kt0; ok && kt < p.kt1; ++kt, ++n_kv) {
        const uint32_t vb = v0 + (n_kv % kStages) * (2 * kOperand >> 4);
        for (int i = 0; i < tiles; ++i) {
          ok = (i > 0 || ready(kVfull, n_kv)) &&
               mbar_wait_bounded(bar + 8 * (kPfull + i), n_p[i] & 1, a.status);
          if (!ok) break;
          ++n_p[i];
          tc_fence_after();
          mma_tmem(tmem + (2 + i) * kTile, tmem + i * kTile, vb, (kt - p.kt0) % kFold != 0);
          if (EXACT) {  // 32 weights' hi, then their lo
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t d = tmem + (2 + i) * kTile, w = tmem + i * kTile + 32 * (k >> 1) + 8 * (k & 1);
              const uint32_t v = vb + k * (2048 >> 4);
              if (k > 0) mma_tmem(d, w, v, 1);
              mma_tmem(d, w + 16, v, 1);
              mma_tmem(d, w, v + (2 * kOperand >> 4), 1);
            }
          } else {
#pragma unroll
            for (int k = 1; k < 8; ++k)
              mma_tmem(tmem + (2 + i) * kTile, tmem + i * kTile + 8 * k, vb + k * (2048 >> 4), 1);
          }
          if (i == tiles - 1) commit(bar + 8 * (kVempty + n_kv % kStages));
          if (kt + 1 < p.kt1) {
            ok = i > 0 || ready(kKfull, n_kv + 1);
            if (!ok) break;
            scores(i, (n_kv + 1) % kStages);
            if (i == tiles - 1) commit(bar + 8 * (kKempty + (n_kv + 1) % kStages));
          } else {
            commit(bar + 8 * (kOfull + i));
          }
        }
      }
    }
    // nothing of this CTA is in flight when its TMEM and shared memory go
    commit(bar + 8 * kDrain);
    mbar_wait_bounded(bar + 8 * kDrain, 0, a.status);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

// Joins the parts of items that several CTAs shared, in order: a CTA per 8 ROWS rows
// of a KV head, a thread per four dimensions (8 rows of four dimensions are a line of a
// part) of ROWS rows, the loads of PARTS parts in flight together.
template <class OutT, int ROWS, int PARTS>
__global__ void __launch_bounds__(256) kv4_attn_join_kernel(Kv4AttnArgs a, int groups) {
  const int lane = threadIdx.x & 31;
  const int rg = blockIdx.x % groups, h = blockIdx.x / groups % a.n_kv;
  const int b = blockIdx.x / groups / a.n_kv;
  pdl_wait_then_release();
  const long long *plan = reinterpret_cast<const long long *>(a.plan);
  const long long quota = plan[0], first = plan[1 + b];
  int len, count;
  seq_shape(a, b, len, count);
  const int row0 = rg * 8 * ROWS, rt = row0 / kRows;
  if (row0 >= count * a.group) return;
  const int nkt = key_tiles(len, count, a.group, rt);
  if (nkt == 0) return;
  long long before = 0;
  for (int k = lane; k < rt; k += 32) before += key_tiles(len, count, a.group, k);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  const long long x = first + before * a.n_kv + (long long)h * nkt;
  const int c0 = (int)(x / quota), c1 = (int)((x + nkt - 1) / quota);
  if (c0 == c1) return;
  const int r = row0 - rt * kRows + (threadIdx.x & 7), c4 = threadIdx.x >> 3;
  auto part_of = [&](int c) { return a.parts + ((size_t)c * 2 + (c == c0 ? 1 : 0)) * kPartFloats; };
  float top[ROWS], sum[ROWS] = {};
  float4 v[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    top[i] = -INFINITY;
    v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll 1
  for (int c = c0; c <= c1; c += PARTS) {
    float4 o[PARTS][ROWS];
    float m[PARTS][ROWS], l[PARTS][ROWS];
#pragma unroll
    for (int k = 0; k < PARTS; ++k) {
      const float *p = part_of(min(c + k, c1));
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        o[k][i] = reinterpret_cast<const float4 *>(p)[c4 * kRows + r + 8 * i];
        m[k][i] = p[kRows * kKv4D + r + 8 * i];
        l[k][i] = p[kRows * (kKv4D + 1) + r + 8 * i];
      }
    }
#pragma unroll
    for (int k = 0; k < PARTS; ++k) {
      if (c + k > c1) break;
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const float4 x = o[k][i];
        const float up = fmaxf(top[i], m[k][i]);
        const float fo = top[i] == up ? 1.f : ex2(top[i] - up),
                    f = m[k][i] == up ? 1.f : ex2(m[k][i] - up);
        v[i].x = fmaf(f, x.x, v[i].x * fo);
        v[i].y = fmaf(f, x.y, v[i].y * fo);
        v[i].z = fmaf(f, x.z, v[i].z * fo);
        v[i].w = fmaf(f, x.w, v[i].w * fo);
        sum[i] = fmaf(f, l[k][i], sum[i] * fo);
        top[i] = up;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int row = rt * kRows + r + 8 * i;
    if (row >= count * a.group) continue;
    const int t = row / a.group;
    const float inv = sum[i] == 0.f ? 0.f : 1.f / sum[i];
    OutT e[4] = {from_float<OutT>(v[i].x * inv), from_float<OutT>(v[i].y * inv),
                 from_float<OutT>(v[i].z * inv), from_float<OutT>(v[i].w * inv)};
    *reinterpret_cast<uint2 *>(reinterpret_cast<OutT *>(a.out) +
                               (((size_t)b * a.tokens + t) * a.n_heads + h * a.group + row -
                                t * a.group) * kKv4D + 4 * c4) = *reinterpret_cast<const uint2 *>(e);
  }
}

template <class OutT>
int many(mlm_ctx *ctx, const Kv4AttnArgs &a) {
  const int st = check_launch_pdl(ctx,
                                  launch_pdl(kv4_attn_many_kernel<OutT>, dim3(ctx->sm_count),
                                             dim3(kThreads), smem_bytes(a.batch), ctx->stream, a),
                                  "mlm_attn_kv4");
  if (st != MLM_OK) return st;
  const int rows = a.tokens * a.group;
  // Short of a CTA per SM the rows have many parts each: 8 rows per CTA, 8 parts at a time
  // (8 tokens at 2000 rows, 32/8 heads: 18.3 us, 28.2 with 32 rows); else 32 rows (1024
  // tokens at 8192: 147 us, 160 with 8)
  const bool few = (long long)((rows + 31) / 32) * a.n_kv * a.batch < ctx->sm_count;
  const int groups = few ? (rows + 7) / 8 : (rows + 31) / 32;
  return check_launch_pdl(
      ctx,
      launch_pdl(few ? kv4_attn_join_kernel<OutT, 1, 8> : kv4_attn_join_kernel<OutT, 4, 2>,
                 dim3((unsigned)groups * a.n_kv * a.batch), dim3(256), 0, ctx->stream, a, groups),
      "mlm_attn_kv4 (join)");
}

}  // namespace

size_t kv4_many_parts_bytes(int sm_count) {
  return sizeof(float) * 2 * sm_count * kPartFloats;
}

int kv4_attn_many_init(mlm_ctx *ctx) {
  MLM_CUDA_TRY(ctx, cudaFuncSetAttribute(kv4_attn_many_kernel<__half>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem_bytes(MLM_KV4_MAX_BATCH)));
  MLM_CUDA_TRY(ctx, cudaFuncSetAttribute(kv4_attn_many_kernel<__nv_bfloat16>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem_bytes(MLM_KV4_MAX_BATCH)));
  return MLM_OK;
}

int kv4_attn_many(mlm_ctx *ctx, const Kv4AttnArgs &a, int out_type) {
  return out_type == MLM_TYPE_F16 ? many<__half>(ctx, a) : many<__nv_bfloat16>(ctx, a);
}

}  // namespace mlm
