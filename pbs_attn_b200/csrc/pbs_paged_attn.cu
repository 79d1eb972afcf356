// Causal attention of new tokens over a paged cache of 16, 8 or 4 bits: out = softmax(scale q K^T) V in one pass over the cache.
//
// Mathematics.  With values of 4 bits K = lo + code * step (step and lo per token and group g of channels)
//   q . k_t  =  sum_g  step_{t,g} (q_g . code_{t,g})  +  lo_{t,g} sum(q_g)
//   o_d      =  sum_t (p_t step_{t,g}) code_{t,d}  +  sum_t p_t lo_{t,g},         g the group of channel d,
// so the codes themselves go into the matrix products and steps and minima act on sums (K) or on the weights (V).  A code's four bits,
// masked out of a word of eight, ARE an fp16 number: bits 0-3 of a half are code * 2^-24 and bits 4-7 code * 2^-20, subnormal numbers that the
// tensor cores multiply exactly.  A word of eight codes costs four ANDs and a shift to become four operand registers, and the factors
// 2^24 and 1/16 go into the queries and the final sums.
//
// With values of 8 bits K = code * scale, V too (a scale for a block of 16 to 64 tokens, so one for the 16 of a product)
//   q . k_t  =  scale_t (q . code_t),        o_d  =  sum_t (p_t scale_t) code_{t,d}.
// K's codes go into the tensor cores as the bytes that they are, m16n8k32, against queries of two bytes (high and low, two products whose sum
// is that of integers): nothing is unpacked.  V's codes must meet weights, which have no two bytes' range, so a byte plus 128, a subnormal
// fp16 number by its bits, meets fp16 weights, and one more product of 128 and the weights, for all channels, is what the sums are less.  In
// fp16 what the rounding of the weights left is a second product: 73 us for 20 queries a head (16 sequences of 2000 to 8192) where one takes 69, no
// difference for 8 queries.
//
// What bounds it: the cache is read once, 2 D bytes a token and KV head in 8 bits and (D + 8 D / G) in 4, and a step of the batch has few queries a
// head, so HBM bounds long caches and latency short ones.  Tokens are the rows (M) of both products and the queries of a KV head the
// columns (N = 8 NT), because a group of 8 or fewer queries then fills an m16n8k16 product; with queries as rows half of it would be
// padding.  mma.sync and not tcgen05: the operand that changes is unpacked in registers, tcgen05 would take it back through shared
// memory (four times the bytes that came in), and the tensor cores are far from being the limit.
//
// Work is cut by tokens, not by sequences: all (sequence, row tile, KV head) items in a row, in units of a tile a warp, are dealt
// to the resident CTAs in equal contiguous shares, so lengths may differ at will and nothing about them has to be known on the host.
// Items that several CTAs share are joined by all of them together, once each has written its partial result (they wait for one another, so
// the grid is launched cooperatively): each joins its part of the rows, from the partial results in the order of the CTAs: same bits every time.
// (With the last CTA of an item joining all of it, one SM read up to 256 KB while the others were done: 5 us instead of 3.)
//
// Measured (B200, GPU time): 64 sequences of 12000 to 16384, 8 KV heads of 128, groups of 64, bf16: 207 us for 1.05 GB, 5.1 TB/s, 77 % of the copy
// rate; 231 us and 69 % under load for seconds, when the power cap lowers the clock.  (The copies alone take 164 us, the arithmetic alone 172: 575
// instructions for 32 tokens, half of them on the ALU pipe.)  One sequence of 131072: 41 us, 3.7 TB/s; of 32768 with 4 KV heads: 13 us.  Several
// queries a head make it arithmetic: 20 (64 sequences of up to 4096) run at 25 % of the copy rate, 32 (8 of up to 8192) at 15; 8 heads of 64
// channels at 38, two of 256 at 30.  Pages of 16 bits, 64 sequences of up to 4096: 121 us for 0.8 GB, the copy rate, under load too; one of
// 131072: 89 us, 92 %; 20 queries a head, 8 of up to 8192: 38 us, 67 %.  8 bits, 64 sequences of 12000 to 16384: 328 us for 1.86 GB, 86 % of the
// copy rate, 336 under load (318 instructions for 16 tokens; with both products in fp16, codes less 1152 by an instruction each, 429, 327 us and 386
// under load); one of 131072: 56 us, 73 %; 64 of 2000 to 4096: 75 us, 81 %; 16 of 2000 to 4096 with 8, 16 and 32 queries a head 52, 39 and 27 %.
//
// Within a CTA every warp takes every eighth (fourth) tile of 16 or 32 tokens through its own ring of cp.async stages, with its own running
// reference and sums; warps meet once an item.
#include <atomic>
#include <climits>
#include <type_traits>

#include "pbs_paged.cuh"

namespace pbs {
namespace {

constexpr int kMaxBatch = 4096, kMaxGrid = PBS_PAGED_COUNTER_BYTES / 8;

// Limit of the wait for an item's parts, and the hook that makes it run out (pbs_debug_set_attn_wait).
std::atomic<unsigned long long> g_wait_ns{2000000000ull};
std::atomic<int> g_drop_arrive{0};

template <int DT_, int D_, int BITS_, int G_, int NT_>
struct Cfg {
  static constexpr int DT = DT_, D = D_, BITS = BITS_, G = G_, NT = NT_;
  using T = typename Elem<DT>::T;
  static constexpr int COLS = 8 * NT;                              // queries of a tile
  static constexpr int MT = BITS == 4 && NT <= 2 && NT * D <= 256 ? 2 : 1;   // 16-token products a tile, as registers allow
  static constexpr int TILE = 16 * MT;
  static constexpr int WARPS = BITS == 16 && D == 256 ? 4 : 8;
  static constexpr int THREADS = 32 * WARPS;
  static constexpr int UNIT = WARPS * TILE;                        // tokens that work is dealt in
  static constexpr int ROW = D * BITS / 8;                         // bytes of a token's row
  static constexpr int CH = ROW / 16;
  static constexpr int NG = BITS == 4 ? D / G : 1;
  static constexpr int PROW = BITS == 4 ? 4 * NG : 0;
  static constexpr int SCALES = BITS == 8 ? 16 : 0;                // bytes of a tile's scales: of keys and of values, for each 16 tokens
  static constexpr int STAGE = TILE * 2 * (ROW + PROW) + SCALES;
  // CTAs a SM: two where registers allow (8 bits, two tiles of queries of 64 channels: 26 us against 31; of 128, spilling a little: no difference)
  static constexpr int OCC = BITS == 8 ? NT * D <= 128 ? 2 : 1 : BITS == 4 && NT == 1 && D <= 128 ? 2 : 1;
  // (with two CTAs a SM a third stage of 128 channels gained nothing: 64 sequences of 16384 205 us with it, 203 without; and the batch's
  // prefix sums have room)
  static constexpr int BUDGET = (OCC == 2 ? BITS == 8 ? 97 : 96 : 200) * 1024;
  static constexpr int STAGES_FIT = BUDGET / (WARPS * STAGE);
  static constexpr int STAGES = STAGES_FIT < 2 ? 2 : STAGES_FIT > 4 ? 4 : STAGES_FIT;
  static constexpr int RING = WARPS * STAGES * STAGE;
  static constexpr int OROW = D + 4;                               // floats of a row of partial sums: four on, so that stores spread over the banks
  static constexpr int MERGE = WARPS * COLS * (OROW + 2) * 4;
  static constexpr int POOL = RING > MERGE ? RING : MERGE;
  static constexpr bool FAR = BITS != 16 && DT == PBS_BF16;        // references may lie 2^170 apart (see factor_of)
  static constexpr bool REST = BITS == 8 && DT == PBS_FP16;        // weights are held in two fp16 numbers (see Warp::tile)
  static constexpr bool LESS8 = BITS == 4 && DT == PBS_FP16;       // V's products are of code - 8 (see Warp)
  static constexpr int SHIFT = BITS == 4 && !LESS8 ? WARPS * COLS * NG * 4 : 0;
  static constexpr int QFRAG = COLS * D * 2;
  static constexpr int FIXED = POOL + QFRAG + SHIFT + COLS * NG * 4 + COLS * 8;      // then the batch's prefix sums
  static_assert(FIXED + kMaxBatch * 4 + 256 <= 227 * 1024, "shared memory");
};

struct AttnArgs {
  PagedArgs a;
  RowTensor q, out;
  // steps from page to page and from slot to slot: rows in 16 bytes, params in 4, so that 32 bits hold every offset in a pool
  uint32_t k_page, k_slot, v_page, v_slot, kp_page, kp_slot, vp_page, vp_slot;
  int dense;                                                       // a page's rows of a head lie together, its params too
  int q_heads, group, row_tiles;
  float scale;                                                     // times log2(e)
  int drop_arrive;                                                 // diagnostic: CTA 0 does not count its part
  unsigned long long wait_ns;
  unsigned* counters;                                              // by the first CTA of an item: parts written, and CTAs that have seen all of them
  float* partials;                                                 // [CTA][2]: COLS x D sums, COLS references, COLS sums of weights
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Copies N bytes, or fills them with zeros.
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool there) {
  const int n = there ? N : 0;
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(n) : "memory");
}
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load_matrices_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// kind: PBS_BF16 or PBS_FP16
template <int KIND>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (KIND == PBS_BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <class T>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) return pack_half(a, b);
  else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// Integers: 16 x 32 signed bytes times 32 x 8.
__device__ __forceinline__ void mma_bytes(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Signed bytes 0 and 2, or 1 and 3, of a word, plus 128 and times 2^-24: fp16 numbers by their bits.
__device__ __forceinline__ uint32_t bytes02(uint32_t w) { return (w & 0x00ff00ffu) ^ 0x00800080u; }
__device__ __forceinline__ uint32_t bytes13(uint32_t w) { return __byte_perm(w, 0, 0x4341) ^ 0x00800080u; }
// Step (low half) and minimum (high half) of a word of params.
template <class T>
__device__ __forceinline__ float step_of(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)w));
  else return __uint_as_float(w << 16);
}
template <class T>
__device__ __forceinline__ float low_of(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)(w >> 16)));
  else return __uint_as_float(w & 0xffff0000u);
}

// The larger step and the minimum of larger magnitude of two words of params (NaN gives way).
template <class T>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __hmax2(*reinterpret_cast<const __half2*>(&a), __habs2(*reinterpret_cast<const __half2*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), __habs2(*reinterpret_cast<const __nv_bfloat162*>(&b)));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// 16-byte piece `ch` of row `row` in shared memory: neighbouring rows' pieces lie in different banks, so eight rows are read at once.
template <class C>
__device__ __forceinline__ int piece(int row, int ch) {
  constexpr int PER = C::CH >= 8 ? 1 : 8 / C::CH, MASK = (C::CH >= 8 ? 8 : C::CH) - 1;
  return row * C::ROW + ((ch ^ ((row / PER) & MASK)) << 4);
}

// Brings sums from one reference to another, whose difference is d.  References of bf16 caches of 8 and 4 bits differ with the steps, too, up to 2^170, while
// the sums of weights that they are for are of one size: the factor is applied as its root, twice.
template <class C>
__device__ __forceinline__ float factor_of(float d) { return exp2_fast(C::FAR ? 0.5f * d : d); }
template <class C>
__device__ __forceinline__ float scaled(float x, float f) { return C::FAR ? x * f * f : x * f; }
template <class C>
__device__ __forceinline__ float add_scaled(float f, float x, float sum) { return fmaf(f, C::FAR ? x * f : x, sum); }

// Params of one token, NG words.
template <class C>
__device__ __forceinline__ void load_params(uint32_t (&w)[C::NG], const uint8_t* p) {
  if constexpr (C::NG == 1) w[0] = *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (C::NG == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x; w[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < C::NG; i += 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(p + 4 * i);
      w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
    }
  }
}

// One warp's running attention of COLS queries.
//
// Weights are p = 2^(score - ref) with a reference per query that is raised only when a product p * step could leave fp16's range (above
// 2^15), to where the largest is 2^7: so the maximum over the warp is taken once in a while and not every tile, and the products, which
// are what the result is made of, keep 2^21 below the largest before they lose bits.
//
// Sums of V's codes as they are grow with the number of tokens, while in flat attention what they leave beside the minima shrinks with its
// root; what the tensor cores cut off such sums then shows (8 sequences of 131072: relative error 5.2e-3).  So
//   fp16: each product is followed by one of -8 with the same weights, and the minimum moves up by 8 steps; a weight's rounding, too, acts on
//         code - 8 then and not on the code (3.1e-4, of which the result's own rounding is 2.1e-4);
//   bf16: every kShiftEvery tiles the sums are moved by what one of each group's has come to, and that is kept aside (1.7e-3, the result's
//         own rounding).  The other way costs 10 % of the time where it goes into arithmetic, this one 1.
//
// 8 bits: every kShiftEvery tiles the sums are made less what 128 and the weights, as they were rounded, have come to: what is left is that of the
// codes, and rounded weights act on code and not on code + 128.  Within eight tiles the larger sums cost up to 2^-12 of a
// code (1.9e-4 of the weighted scales in 9000 calls of all sizes): a 2000th of what writing a value did.
//
// In bf16 a minimum may be much larger than any step (a group of equal values has none), up to 2^128, and 32 bits hold its products with weights if
// it counts as a step of 2^-64 of it: they stay below 2^79.
//
// 16 bits: what a weight meets is a value of the type.  In fp16 that is up to 2^16 and 32 bits have room for it; bf16's values go up to 2^128, so its
// weights, which are bf16 themselves, are kept 2^40 smaller: 2^25 tokens of the largest value and weight add up to less than 2^128.
constexpr int kShiftEvery = 8;
constexpr int kWhole = 2;                                          // units of sequences that are not split

template <class C>
struct Warp {
  using T = typename C::T;
  static constexpr int kRoom = C::BITS == 16 && C::DT == PBS_BF16 ? 40 : 0;        // powers of 2 that weights are kept smaller by
  float o[C::D / 16][C::NT][4];
  float om[C::BITS == 4 ? C::NG : 1][C::NT][2];                    // sums of p * lo, this lane's tokens
  [[maybe_unused]] float o128[C::BITS == 8 ? C::NT : 1][4];        // 8 bits: what o has to be less
  float l[C::NT][2], ref[C::NT][2];
  const uint4* qf;                                                 // this lane's query fragments, C::NT * 32 apart from chunk to chunk
  const float* qsum;
  const float* factor;
  const int* limit;
  float* shift;                                                    // bf16: what sums were moved by, [group][query]
  int lane;

  __device__ __forceinline__ void start() {
    if constexpr (C::SHIFT > 0) {
      for (int i = lane; i < C::NG * C::COLS; i += 32) shift[i] = 0.f;
      __syncwarp();
    }
    if constexpr (C::BITS == 8) {
#pragma unroll
      for (int n = 0; n < C::NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) o128[n][c] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < C::D / 16; ++i)
#pragma unroll
      for (int n = 0; n < C::NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[i][n][c] = 0.f;
#pragma unroll
    for (int n = 0; n < C::NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        l[n][c] = 0.f;
        ref[n][c] = -CUDART_INF_F;
#pragma unroll
        for (int g = 0; g < (C::BITS == 4 ? C::NG : 1); ++g) om[g][n][c] = 0.f;
      }
  }

  // Scores of the tile (times 2^-k of the query's scaling: `factor` has the rest): tot[m][n] holds tokens lane / 4 and + 8, queries 2 (lane % 4) and + 1
  __device__ __forceinline__ void scores(float (&tot)[C::MT][C::NT][4], const uint8_t* stage) const {
    const uint32_t k_at = smem_addr(stage);
    const int row = lane & 15, half = lane >> 4;
#pragma unroll
    for (int m = 0; m < C::MT; ++m)
#pragma unroll
      for (int n = 0; n < C::NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) tot[m][n][c] = 0.f;
    if constexpr (C::BITS == 16) {
#pragma unroll
      for (int ks = 0; ks < C::D / 16; ++ks) {
        uint32_t r[C::MT][4];
#pragma unroll
        for (int m = 0; m < C::MT; ++m) load_matrices(r[m], k_at + piece<C>(16 * m + row, 2 * ks + half));
#pragma unroll
        for (int n = 0; n < C::NT; ++n) {
          const uint4 q = qf[(ks / 2 * C::NT + n) * 32];
#pragma unroll
          for (int m = 0; m < C::MT; ++m) mma<C::DT>(tot[m][n], r[m][0], r[m][1], r[m][2], r[m][3], ks % 2 ? q.z : q.x, ks % 2 ? q.w : q.y);
        }
      }
    } else if constexpr (C::BITS == 8) {
      int high[C::MT][C::NT][4], low[C::MT][C::NT][4];             // with the queries' high and low bytes
#pragma unroll
      for (int m = 0; m < C::MT; ++m)
#pragma unroll
        for (int n = 0; n < C::NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) high[m][n][c] = low[m][n][c] = 0;
#pragma unroll
      for (int j = 0; j < C::CH / 2; ++j) {
        uint32_t r[C::MT][4];
#pragma unroll
        for (int m = 0; m < C::MT; ++m) load_matrices(r[m], k_at + piece<C>(16 * m + row, 2 * j + half));
#pragma unroll
        for (int n = 0; n < C::NT; ++n) {
          const uint4 q = qf[(j * C::NT + n) * 32];
#pragma unroll
          for (int m = 0; m < C::MT; ++m) {
            mma_bytes(high[m][n], r[m], q.x, q.y);
            mma_bytes(low[m][n], r[m], q.z, q.w);
          }
        }
      }
#pragma unroll
      for (int m = 0; m < C::MT; ++m)
#pragma unroll
        for (int n = 0; n < C::NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) tot[m][n][c] = (float)(high[m][n][c] * 256 + low[m][n][c]);
    } else {
      uint32_t kp[C::MT][2][C::NG];
      const uint8_t* params = stage + 2 * C::TILE * C::ROW;
#pragma unroll
      for (int m = 0; m < C::MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) load_params<C>(kp[m][h], params + (16 * m + lane / 4 + 8 * h) * C::PROW);
      float acc[C::MT][C::NT][4];
#pragma unroll
      for (int j2 = 0; j2 < C::CH / 2; ++j2) {
        uint32_t r[C::MT][4];
#pragma unroll
        for (int m = 0; m < C::MT; ++m) load_matrices(r[m], k_at + piece<C>(16 * m + row, 2 * j2 + half));
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
          const int j = 2 * j2 + jj;
          if (j * 32 % C::G == 0) {
#pragma unroll
            for (int m = 0; m < C::MT; ++m)
#pragma unroll
              for (int n = 0; n < C::NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[m][n][c] = 0.f;
          }
          constexpr uint32_t M0 = 0x000f000fu, M1 = 0x00f000f0u;
#pragma unroll
          for (int n = 0; n < C::NT; ++n) {
            const uint4 q = qf[(j * C::NT + n) * 32];
#pragma unroll
            for (int m = 0; m < C::MT; ++m) {
              const uint32_t x = r[m][2 * jj], y = r[m][2 * jj + 1], x8 = x >> 8, y8 = y >> 8;
              mma<PBS_FP16>(acc[m][n], x & M0, y & M0, x & M1, y & M1, q.x, q.y);
              mma<PBS_FP16>(acc[m][n], x8 & M0, y8 & M0, x8 & M1, y8 & M1, q.z, q.w);
            }
          }
          if ((j + 1) * 32 % C::G == 0) {
            const int g = j * 32 / C::G;
#pragma unroll
            for (int n = 0; n < C::NT; ++n) {
              const float2 s = *reinterpret_cast<const float2*>(qsum + g * C::COLS + 8 * n + 2 * (lane % 4));
#pragma unroll
              for (int m = 0; m < C::MT; ++m)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                  tot[m][n][c] = fmaf(acc[m][n][c], step_of<T>(kp[m][c / 2][g]), fmaf(low_of<T>(kp[m][c / 2][g]), c % 2 ? s.y : s.x, tot[m][n][c]));
            }
          }
        }
      }
    }
  }

  // What the weights of tokens meet, for the largest of their steps and minima; at least `least`, for weights to stay below 2^85.
  static __device__ __forceinline__ constexpr float least() { return C::DT == PBS_BF16 ? 0x1p-70f : 0x1p-40f; }
  static __device__ __forceinline__ float met(uint32_t w) {
    if constexpr (C::BITS == 8) return fmaxf(fabsf(__uint_as_float(w)), least());
    if constexpr (C::DT == PBS_BF16) return fmaxf(fmaxf(step_of<T>(w), low_of<T>(w) * 0x1p-64f), least());
    else return fmaxf(step_of<T>(w), least());
  }

  static __device__ __forceinline__ bool too_large(float weight, float wide, float ref) {
    return !(weight * wide <= 32768.f) || ref == -CUDART_INF_F;
  }

  // Raises the references of the queries that need it to the largest product of this tile (x: scores, in powers of 2; wide: the most that weights
  // of what a query sees meet), and weighs the tile anew.  The largest product and not the largest score and step: a token that hardly weighs
  // must not push the weights of the others, whose steps may be much smaller, out of fp16.
  __device__ __forceinline__ void raise(const float (&x)[C::MT][C::NT][4], float (&p)[C::MT][C::NT][4], const float (&wide)[C::NT][2],
                                        const uint32_t (&vp)[C::MT][2][C::NG]) {
    float meets[C::MT][2];                                         // by token, in powers of 2
#pragma unroll
    for (int m = 0; m < C::MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        meets[m][h] = (float)kRoom;
        if constexpr (C::BITS == 8) meets[m][h] = __log2f(fminf(met(vp[m][0][0]), 0x1p127f));
        if constexpr (C::BITS == 4) {
          uint32_t w = 0;
#pragma unroll
          for (int g = 0; g < C::NG; ++g) w = larger<T>(w, vp[m][h][g]);
          meets[m][h] = __log2f(fminf(met(w), 0x1p127f));
        }
      }
#pragma unroll
    for (int n = 0; n < C::NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float most = -CUDART_INF_F, weight = 0.f;
#pragma unroll
        for (int m = 0; m < C::MT; ++m) {
          most = fmaxf(most, fmaxf(x[m][n][c] + meets[m][0], x[m][n][c + 2] + meets[m][1]));
          weight = fmaxf(weight, fmaxf(p[m][n][c], p[m][n][c + 2]));
        }
        const uint32_t need = __ballot_sync(0xffffffffu, too_large(weight, wide[n][c], ref[n][c]));
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, s));
        if (!(need & 0x11111111u << lane % 4)) continue;           // (whole columns of lanes agree)
        const float old = ref[n][c];
        if (most > -CUDART_INF_F) ref[n][c] = fmaxf(old, most - 7.f);
        if (ref[n][c] != old && old > -CUDART_INF_F) {             // (before the first reference nothing has been summed up)
          const float keep = factor_of<C>(old - ref[n][c]);
          l[n][c] = scaled<C>(l[n][c], keep);
          if constexpr (C::BITS == 8) o128[n][c] = scaled<C>(o128[n][c], keep);
#pragma unroll
          for (int i = 0; i < C::D / 16; ++i) {
            o[i][n][c] = scaled<C>(o[i][n][c], keep);
            o[i][n][c + 2] = scaled<C>(o[i][n][c + 2], keep);
          }
#pragma unroll
          for (int g = 0; g < (C::BITS == 4 ? C::NG : 1); ++g) {
            om[g][n][c] = scaled<C>(om[g][n][c], keep);
            if (C::SHIFT > 0 && lane < 4) shift[g * C::COLS + 8 * n + 2 * lane + c] = scaled<C>(shift[g * C::COLS + 8 * n + 2 * lane + c], keep);
          }
        }
#pragma unroll
        for (int m = 0; m < C::MT; ++m)
#pragma unroll
          for (int h = 0; h < 4; h += 2) p[m][n][c + h] = x[m][n][c + h] == -CUDART_INF_F ? 0.f : exp2_fast(x[m][n][c + h] - ref[n][c]);
      }
  }

  // Infinities and NaNs among the values of a tile that not all queries see: 0 for the product, and added where they are seen.
  __device__ __forceinline__ void add_not_finite(const uint8_t* v, int t0) {
    for (int t = 0; t < C::TILE; ++t)
#pragma unroll
      for (int i = 0; i < C::D / 16; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int d = 16 * i + lane / 4 + 8 * h;
          const float x = Elem<C::DT>::ld(reinterpret_cast<const T*>(v + piece<C>(t, d / 8)) + d % 8);
          if (fabsf(x) <= 3.402823466e38f) continue;
#pragma unroll
          for (int n = 0; n < C::NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c)
              if (t0 + t < limit[8 * n + 2 * (lane % 4) + c]) o[i][n][2 * h + c] += x;
        }
  }

  __device__ __forceinline__ void move_sums() {
    if constexpr (C::BITS == 8) {
#pragma unroll
      for (int n = 0; n < C::NT; ++n) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int i = 0; i < C::D / 16; ++i) {
            o[i][n][c] -= o128[n][c];
            o[i][n][c + 2] -= o128[n][c];
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) o128[n][c] = 0.f;
      }
    }
    if constexpr (C::SHIFT > 0) {
#pragma unroll
      for (int g = 0; g < C::NG; ++g)
#pragma unroll
        for (int n = 0; n < C::NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            constexpr int TILES = C::G / 16;                       // of 16 channels, in a group
            const float x = __shfl_sync(0xffffffffu, o[g * TILES][n][c], lane % 4);
#pragma unroll
            for (int i = g * TILES; i < (g + 1) * TILES; ++i) {
              o[i][n][c] -= x;
              o[i][n][c + 2] = fmaf(-17.f, x, o[i][n][c + 2]);     // (low + 16 high)
            }
            if (lane < 4) shift[g * C::COLS + 8 * n + 2 * lane + c] += x;
          }
    }
  }

  // Takes in the tile of tokens t0 .. in shared memory.  MASKED: some query does not see all of them, or 16 of them (a bit of hole) have no page.
  template <bool MASKED>
  __device__ __forceinline__ void tile(const uint8_t* stage, int t0, uint32_t hole) {
    float x[C::MT][C::NT][4], p[C::MT][C::NT][4];
    scores(x, stage);
    [[maybe_unused]] float ks[C::MT];                              // 8 bits: scales of the keys
    if constexpr (C::BITS == 8) {
#pragma unroll
      for (int m = 0; m < C::MT; ++m) ks[m] = *reinterpret_cast<const float*>(stage + 2 * C::TILE * C::ROW + 8 * m);
    }
    bool seen[C::MT][C::NT][4];
#pragma unroll
    for (int n = 0; n < C::NT; ++n) {
      const float2 f_all = *reinterpret_cast<const float2*>(factor + 8 * n + 2 * (lane % 4));
      const int2 lim = MASKED ? *reinterpret_cast<const int2*>(limit + 8 * n + 2 * (lane % 4)) : make_int2(0, 0);
#pragma unroll
      for (int m = 0; m < C::MT; ++m) {
        const float2 f = C::BITS == 8 ? make_float2(f_all.x * ks[m], f_all.y * ks[m]) : f_all;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (MASKED) {
            x[m][n][c] *= c % 2 ? f.y : f.x;
            seen[m][n][c] = t0 + 16 * m + lane / 4 + c / 2 * 8 < (c % 2 ? lim.y : lim.x) && !(hole >> m & 1);
            if (!seen[m][n][c]) x[m][n][c] = -CUDART_INF_F;
            p[m][n][c] = seen[m][n][c] ? exp2_fast(x[m][n][c] - ref[n][c % 2]) : 0.f;
          } else {
            p[m][n][c] = exp2_fast(fmaf(x[m][n][c], c % 2 ? f.y : f.x, -ref[n][c % 2]));
          }
        }
      }
    }
    uint32_t vp[C::MT][2][C::NG];
    float wide[C::NT][2];
    float widest = (float)(1ull << kRoom);
    if constexpr (C::BITS == 4) {
      uint32_t token[C::MT][2], all = 0;
      const uint8_t* params = stage + 2 * C::TILE * C::ROW + C::TILE * C::PROW;
#pragma unroll
      for (int m = 0; m < C::MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          load_params<C>(vp[m][h], params + (16 * m + lane / 4 + 8 * h) * C::PROW);
          token[m][h] = 0;
#pragma unroll
          for (int g = 0; g < C::NG; ++g) token[m][h] = larger<T>(token[m][h], vp[m][h][g]);
          all = larger<T>(all, token[m][h]);
        }
      widest = met(all);
      if constexpr (MASKED) {
#pragma unroll
        for (int n = 0; n < C::NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            wide[n][c] = least();
#pragma unroll
            for (int m = 0; m < C::MT; ++m)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (seen[m][n][2 * h + c]) wide[n][c] = fmaxf(wide[n][c], met(token[m][h]));
          }
      }
    }
    if constexpr (C::BITS == 8) {
      widest = least();
#pragma unroll
      for (int m = 0; m < C::MT; ++m) {
        vp[m][0][0] = *reinterpret_cast<const uint32_t*>(stage + 2 * C::TILE * C::ROW + 8 * m + 4);
        widest = fmaxf(widest, met(vp[m][0][0]));
      }
      if constexpr (MASKED) {
#pragma unroll
        for (int n = 0; n < C::NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            wide[n][c] = least();
#pragma unroll
            for (int m = 0; m < C::MT; ++m)
              if (seen[m][n][c] || seen[m][n][2 + c]) wide[n][c] = fmaxf(wide[n][c], met(vp[m][0][0]));
          }
      }
    }
    bool need = false;
#pragma unroll
    for (int n = 0; n < C::NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (!MASKED || C::BITS == 16) wide[n][c] = widest;
        float weight = 0.f;
#pragma unroll
        for (int m = 0; m < C::MT; ++m) weight = fmaxf(weight, fmaxf(p[m][n][c], p[m][n][c + 2]));
        need = need || too_large(weight, wide[n][c], ref[n][c]);
      }
    if (__any_sync(0xffffffffu, need)) {
      if (!MASKED) {
#pragma unroll
        for (int n = 0; n < C::NT; ++n) {
          const float2 f = *reinterpret_cast<const float2*>(factor + 8 * n + 2 * (lane % 4));
#pragma unroll
          for (int m = 0; m < C::MT; ++m)
#pragma unroll
            for (int c = 0; c < 4; ++c) x[m][n][c] *= C::BITS == 8 ? (c % 2 ? f.y : f.x) * ks[m] : c % 2 ? f.y : f.x;
        }
      }
      raise(x, p, wide, vp);
    }
#pragma unroll
    for (int n = 0; n < C::NT; ++n)
#pragma unroll
      for (int m = 0; m < C::MT; ++m) {
        l[n][0] += p[m][n][0] + p[m][n][2];
        l[n][1] += p[m][n][1] + p[m][n][3];
      }
    const uint8_t* v = stage + C::TILE * C::ROW;
    const uint32_t v_at = smem_addr(v);
    if constexpr (C::BITS == 16) {
      bool clean = true;
      if constexpr (MASKED) {
        constexpr uint32_t E = C::DT == PBS_BF16 ? 0x7f80u : 0x7c00u;
        for (int i = lane; i < C::TILE * C::CH; i += 32) {
          const uint4 w = *reinterpret_cast<const uint4*>(v + 16 * i);
          const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) clean = clean && (u[e] & E) != E && ((u[e] >> 16) & E) != E;
        }
        clean = __all_sync(0xffffffffu, clean);
      }
#pragma unroll
      for (int m = 0; m < C::MT; ++m) {
        uint32_t b[C::NT][2];
#pragma unroll
        for (int n = 0; n < C::NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // rounded to the pages' type, which is what the tensor cores multiply pages of 16 bits by: relative error 2.3e-3 in bf16 and 2.9e-4 in
            // fp16 (8 sequences of 2000 to 8192), where the result's own rounding leaves 1.7e-3 and 2.1e-4
            b[n][h] = transpose8(pack<T>(p[m][n][2 * h], p[m][n][2 * h + 1]));
          }
#pragma unroll
        for (int i = 0; i < C::D / 16; ++i) {
          uint32_t r[4];
          load_matrices_t(r, v_at + piece<C>(16 * m + (lane & 7) + ((lane >> 4) << 3), 2 * i + ((lane >> 3) & 1)));
          if constexpr (MASKED) {
            if (!clean) {
              constexpr uint32_t E = C::DT == PBS_BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if ((r[e] & E) == E) r[e] &= 0xffff0000u;
                if (((r[e] >> 16) & E) == E) r[e] &= 0xffffu;
              }
            }
          }
#pragma unroll
          for (int n = 0; n < C::NT; ++n) mma<C::DT>(o[i][n], r[0], r[1], r[2], r[3], b[n][0], b[n][1]);
        }
      }
      if constexpr (MASKED) {
        if (!clean) add_not_finite(v, t0);
      }
    } else if constexpr (C::BITS == 8) {
#pragma unroll
      for (int m = 0; m < C::MT; ++m) {
        uint32_t b[C::NT][2];
        [[maybe_unused]] uint32_t rest[C::REST ? C::NT : 1][2];
        const float s = __uint_as_float(vp[m][0][0]);
#pragma unroll
        for (int n = 0; n < C::NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // a weight of 0 must not meet a scale that is not finite, of tokens that this query does not see; rounded to fp16, 11 bits, of which a
            // result of bf16, 8 bits, shows nothing; for one of fp16 what the rounding left is multiplied too (relative error 2.1e-4, the result's own
            // rounding, and not 2.8e-4 to 3.2e-4)
            const bool s0 = !MASKED || seen[m][n][2 * h], s1 = !MASKED || seen[m][n][2 * h + 1];
            const float w0 = s0 ? p[m][n][2 * h] * s : 0.f, w1 = s1 ? p[m][n][2 * h + 1] * s : 0.f;
            const uint32_t w = pack_half(w0, w1);
            b[n][h] = transpose8(w);
            if constexpr (C::REST) {
              const float2 rounded = __half22float2(*reinterpret_cast<const __half2*>(&w));
              rest[n][h] = transpose8(pack_half(w0 - rounded.x, w1 - rounded.y));
            }
          }
#pragma unroll
        for (int j2 = 0; j2 < C::CH / 2; ++j2) {
          uint32_t r[4];
          load_matrices_t(r, v_at + piece<C>(16 * m + (lane & 15), 2 * j2 + (lane >> 4)));
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {
            // rows of the product: channels 2 i and 2 i + 1 of 16
            const uint32_t y = r[2 * jj], z = r[2 * jj + 1];
            const uint32_t a0 = bytes02(y), a1 = bytes13(y), a2 = bytes02(z), a3 = bytes13(z);
#pragma unroll
            for (int n = 0; n < C::NT; ++n) {
              mma<PBS_FP16>(o[2 * j2 + jj][n], a0, a1, a2, a3, b[n][0], b[n][1]);
              if constexpr (C::REST) mma<PBS_FP16>(o[2 * j2 + jj][n], a0, a1, a2, a3, rest[n][0], rest[n][1]);
            }
          }
        }
        constexpr uint32_t k128 = 0x00800080u;
#pragma unroll
        for (int n = 0; n < C::NT; ++n) {
          mma<PBS_FP16>(o128[n], k128, k128, k128, k128, b[n][0], b[n][1]);
          if constexpr (C::REST) mma<PBS_FP16>(o128[n], k128, k128, k128, k128, rest[n][0], rest[n][1]);
        }
      }
    } else {
#pragma unroll
      for (int m = 0; m < C::MT; ++m) {
        uint32_t b[C::NT][2];
#pragma unroll
        for (int j2 = 0; j2 < C::CH / 2; ++j2) {
          uint32_t r[4];
          load_matrices_t(r, v_at + piece<C>(16 * m + (lane & 15), 2 * j2 + (lane >> 4)));
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {
            const int j = 2 * j2 + jj;
            if (j * 32 % C::G == 0) {                              // a group's weights
              const int g = j * 32 / C::G;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float s = step_of<T>(vp[m][h][g]), low = C::LESS8 ? fmaf(8.f, s, low_of<T>(vp[m][h][g])) : low_of<T>(vp[m][h][g]);
#pragma unroll
                for (int n = 0; n < C::NT; ++n) {
                  // a weight of 0 must not meet a step or minimum that is not finite, of a token that this query does not see
                  const float p0 = p[m][n][2 * h], p1 = p[m][n][2 * h + 1];
                  const bool s0 = !MASKED || seen[m][n][2 * h], s1 = !MASKED || seen[m][n][2 * h + 1];
                  om[g][n][0] = s0 ? fmaf(p0, low, om[g][n][0]) : om[g][n][0];
                  om[g][n][1] = s1 ? fmaf(p1, low, om[g][n][1]) : om[g][n][1];
                  // rounded to fp16, 11 bits: the codes have 4, the result 8 or 11
                  b[n][h] = transpose8(pack_half(s0 ? p0 * s : 0.f, s1 ? p1 * s : 0.f));
                }
              }
            }
            // rows of the product: the low code of a byte, and the byte (low + 16 high, eight bits that fp16 holds as well): four
            // operations for eight codes, where masking the high ones out takes five
            constexpr uint32_t M0 = 0x000f000fu, M = 0x00ff00ffu;
            [[maybe_unused]] constexpr uint32_t kLess = 0x80088008u, kLess16 = 0x80888088u;          // -8 and -(8 + 16 * 8), times 2^-24
            const uint32_t y = r[2 * jj] & M, z = r[2 * jj + 1] & M, y8 = __byte_perm(r[2 * jj], 0, 0x4341), z8 = __byte_perm(r[2 * jj + 1], 0, 0x4341);
#pragma unroll
            for (int n = 0; n < C::NT; ++n) {
              mma<PBS_FP16>(o[2 * j][n], y & M0, y, z & M0, z, b[n][0], b[n][1]);
              if constexpr (C::LESS8) mma<PBS_FP16>(o[2 * j][n], kLess, kLess16, kLess, kLess16, b[n][0], b[n][1]);
              mma<PBS_FP16>(o[2 * j + 1][n], y8 & M0, y8, z8 & M0, z8, b[n][0], b[n][1]);
              if constexpr (C::LESS8) mma<PBS_FP16>(o[2 * j + 1][n], kLess, kLess16, kLess, kLess16, b[n][0], b[n][1]);
            }
          }
        }
      }
    }
  }

  // Sums, reference and weights' sum of this warp's tokens to shared memory, query by query.
  __device__ __forceinline__ void put(float* sums, float* refs, float* weights) {
    __syncwarp();
    if constexpr (C::BITS == 8) move_sums();
#pragma unroll
    for (int n = 0; n < C::NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = 8 * n + 2 * (lane % 4) + c;
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) {
          l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], s);
          if constexpr (C::BITS == 4) {
#pragma unroll
            for (int g = 0; g < C::NG; ++g) om[g][n][c] += __shfl_xor_sync(0xffffffffu, om[g][n][c], s);
          }
        }
        if (lane < 4) {
          refs[col] = ref[n][c];
          weights[col] = l[n][c];
        }
        float* row = sums + col * C::OROW;
        if constexpr (C::BITS == 4) {
#pragma unroll
          for (int j = 0; j < C::CH; ++j) {
            const int g = j * 32 / C::G;
            const float (&e)[4] = o[2 * j][n], (&f)[4] = o[2 * j + 1][n];
            float low = om[g][n][c];
            if constexpr (C::SHIFT > 0) low = fmaf(shift[g * C::COLS + col], 0x1p24f, low);
            *reinterpret_cast<float4*>(row + 32 * j + 4 * (lane / 4)) =
                make_float4(fmaf(e[c], 0x1p24f, low), fmaf(e[c + 2] - e[c], 0x1p20f, low), fmaf(f[c], 0x1p24f, low), fmaf(f[c + 2] - f[c], 0x1p20f, low));
          }
        } else if constexpr (C::BITS == 8) {
#pragma unroll
          for (int i = 0; i < C::D / 16; ++i) *reinterpret_cast<float2*>(row + 16 * i + 2 * (lane / 4)) = make_float2(o[i][n][c] * 0x1p24f, o[i][n][c + 2] * 0x1p24f);
        } else {
#pragma unroll
          for (int i = 0; i < C::D / 16; ++i) {
            row[16 * i + lane / 4] = o[i][n][c];
            row[16 * i + lane / 4 + 8] = o[i][n][c + 2];
          }
        }
      }
  }
};

// Quotients of numbers from 0 by one that does not change: the common ones are small and take an eighth of a division's time.
struct Divisor {
  int d;
  float inverse;
  __device__ __forceinline__ explicit Divisor(int n) : d(n), inverse(1.f / (float)n) {}
  __device__ __forceinline__ int of(int a, int& rest) const {
    int q = (int)((float)a * inverse);
    rest = a - q * d;
    for (; rest < 0; rest += d) --q;
    for (; rest >= d; rest -= d) ++q;
    return q;
  }
  __device__ __forceinline__ int of(int a) const {
    int rest;
    return of(a, rest);
  }
};

// The part of an item that a CTA works on.
struct Item {
  int seq, head, row0;                                             // row = new token * group + query head within the KV head
  int len, full, n;                                                // tokens of the sequence that its row of the table holds, all of them, new ones
  int first, end;                                                  // tokens that the first of the rows sees, and the last
  int unit1;                                                       // the unit behind the item
};

// Brings the queries of an item into the order of the product's second operand (in 8 and 4 bits scaled by a power of two to a maximum in
// [2^14, 2^15), which fp16 holds to 2^-38 of it), and what belongs to each.
template <class C>
struct Queries {
  using T = typename C::T;
  static constexpr int PIECES = C::D / 8, EACH = (C::COLS * PIECES + C::THREADS - 1) / C::THREADS;     // 16-byte pieces of a row; of a thread
  uint4 raws[EACH];

  __device__ __forceinline__ void load(const AttnArgs& p, const Item& it, const Divisor& group) {
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      const int e = threadIdx.x + u * C::THREADS, col = e / PIECES, pc = e % PIECES;
      int h;
      const int i = group.of(it.row0 + col, h);
      raws[u] = make_uint4(0, 0, 0, 0);
      if (e < C::COLS * PIECES && i < it.n)
        raws[u] = *reinterpret_cast<const uint4*>((const T*)p.q.p + it.seq * p.q.st.b + (it.head * p.group + h) * p.q.st.h + i * p.q.st.s + 8 * pc);
    }
  }

  __device__ __forceinline__ void put(const AttnArgs& p, const Item& it, const Divisor& group, uint8_t* frag, float* qsum, float* factor, int* limit) const {
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      const int e = threadIdx.x + u * C::THREADS;
      if (e >= C::COLS * PIECES) break;                              // (whole warps: shuffles are among the lanes of a row)
      const int col = e / PIECES, pc = e % PIECES, i = group.of(it.row0 + col);
      const bool valid = i < it.n;
      const uint4 raw = raws[u];
      float f = p.scale;
      if constexpr (C::BITS == 16) {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int t = 0; t < 4; ++t)
          *reinterpret_cast<uint32_t*>(frag + (((pc / 4) * C::NT + col / 8) * 32 + (col % 8) * 4 + t) * 16 + (pc / 2 % 2 * 2 + pc % 2) * 4) = w[t];
      } else {
        const T* raw8 = reinterpret_cast<const T*>(&raw);
        float x[8], most = 0.f, sum = 0.f;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          x[t] = Elem<C::DT>::ld(raw8 + t);
          most = fmaxf(most, fabsf(x[t]));
        }
#pragma unroll
        for (int s = PIECES / 2; s > 0; s >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, s));
        // most = 2^e * [1, 2): scaled by 2^k, k = 14 - e, kept where 2^k and the factor 2^-k or 2^(24 - k) are ordinary numbers
        int k = most > 0.f ? 14 - ((int)(__float_as_uint(most) >> 23) - 127) : 0;
        if constexpr (C::BITS == 8) {                                // (two signed bytes hold up to 32639)
          if ((__float_as_uint(most) & 0x7fffffu) > 0x7efe00u) --k;
        }
        k = min(max(k, C::BITS == 8 ? -114 : -90), 120);
        const float up = __uint_as_float((uint32_t)(k + 127) << 23);
        f *= __uint_as_float((uint32_t)((C::BITS == 4 ? 24 : 0) - k + 127) << 23);
        if constexpr (C::BITS == 8) {
          // integers of two bytes: rounded by up to 2^-15 of the row's largest, which moves a score by as much of it times the sum of a key's
          // magnitudes at most (bf16 queries lose nothing down to 2^-7 of the largest).  What no integer is makes the row NaN
          uint32_t high[2] = {0, 0}, low[2] = {0, 0};
          float none = 0.f;
#pragma unroll
          for (int t = 0; t < 8; ++t) none += x[t] * 0.f;
#pragma unroll
          for (int s = PIECES / 2; s > 0; s >>= 1) none += __shfl_xor_sync(0xffffffffu, none, s);
          f += none;
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            const int i = __float2int_rn(x[t] * up), h = (i + 128) >> 8;
            high[t / 4] |= (h & 0xff) << t % 4 * 8;
            low[t / 4] |= ((i - h * 256) & 0xff) << t % 4 * 8;
          }
          uint32_t* const at = reinterpret_cast<uint32_t*>(frag + (((pc / 4) * C::NT + col / 8) * 32 + (col % 8) * 4 + pc % 2 * 2) * 16) + pc / 2 % 2;
          at[0] = high[0];
          at[2] = low[0];
          at[4] = high[1];
          at[6] = low[1];
        } else {
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            x[t] = __half2float(__float2half_rn(x[t] * up));
            sum += x[t];
          }
#pragma unroll
          for (int s = C::G / 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
          if (pc % (C::G / 8) == 0) qsum[pc / (C::G / 8) * C::COLS + col] = sum * 0x1p-24f;
          // codes i and i + 4 of a word meet in one register; those of bits 4-7 are 16 times too large
          *reinterpret_cast<uint4*>(frag + (((pc / 4) * C::NT + col / 8) * 32 + (col % 8) * 4 + pc % 4) * 16) =
              make_uint4(pack_half(x[0], x[4]), pack_half(x[1] * 0.0625f, x[5] * 0.0625f), pack_half(x[2], x[6]), pack_half(x[3] * 0.0625f, x[7] * 0.0625f));
        }
      }
      if (pc == 0) {
        factor[col] = f;
        limit[col] = valid ? max(0, min(it.len, it.full - it.n + i + 1)) : INT_MAX;
      }
    }
  }
};

template <class C>
__global__ void __launch_bounds__(C::THREADS, C::OCC) paged_attn_kernel(const __grid_constant__ AttnArgs p) {
  using T = typename C::T;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* frag = smem + C::POOL;
  float* qsum = reinterpret_cast<float*>(frag + C::QFRAG + C::SHIFT);
  float* factor = qsum + C::COLS * C::NG;
  int* limit = reinterpret_cast<int*>(factor + C::COLS);
  int* prefix = limit + C::COLS;                                   // units before sequence b
  __shared__ int scan[C::WARPS];
  __shared__ int arrived;
  const pbs_paged_cache_t& c = p.a.c;
  const pbs_paged_batch_t& bt = p.a.b;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int table_tokens = bt.max_pages << p.a.shift;
  after_the_kernel_before();

  // 8 bits: where all sequences are short (two units at most) a unit is a whole one.  What splitting it saves on a tile goes on joining the parts:
  // 187 tokens take 6.9 us in two units a head, 5.9 in one (500 tokens 7.5 in four, 10.8 in one).
  static_assert((C::UNIT & (C::UNIT - 1)) == 0, "units are a power of two");
  int unit_tokens = C::UNIT;
  const int own_len = tid < bt.batch ? bt.seq_lens[tid] : 0;       // (of up to THREADS sequences all that is read of the lengths here)
  if constexpr (C::BITS == 8) {
    // (as far as their rows of the table go: with a table that short the CTAs are not launched to wait for one another, so nothing may be split)
    bool any = min(own_len, table_tokens) > kWhole * C::UNIT;
    for (int b = tid + C::THREADS; b < bt.batch; b += C::THREADS) any = any || min(bt.seq_lens[b], table_tokens) > kWhole * C::UNIT;
    if (!__syncthreads_or(any)) unit_tokens = kWhole * C::UNIT;
  }
  const int unit_shift = __ffs(unit_tokens) - 1;
  // units of all sequences (an empty one has a unit too: its rows are written)
  const int per = p.row_tiles * c.kv_heads;
  int total = 0;
  for (int b0 = 0; b0 < bt.batch; b0 += C::THREADS) {
    const int b = b0 + tid;
    int u = 0;
    if (b < bt.batch) {
      const int len = b0 == 0 ? own_len : bt.seq_lens[b];
      if (len > table_tokens) paged_fault(p.a, PBS_PAGED_BAD_LENGTH);
      u = max(1, (max(0, min(len, table_tokens)) + unit_tokens - 1) >> unit_shift) * per;
    }
    int sum = u;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, sum, s);
      if (lane >= s) sum += y;
    }
    if (lane == 31) scan[warp] = sum;
    __syncthreads();
    int before = total;
#pragma unroll
    for (int w = 0; w < C::WARPS; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    if (b < bt.batch) prefix[b] = before + sum - u;
    __syncthreads();
  }
  const int share = (total + gridDim.x - 1) / gridDim.x;
  const Divisor by_share(share), by_group(p.group);
  int unit = min(total, (int)blockIdx.x * share);
  const int unit_end = min(total, unit + share);

  Warp<C> w;
  w.lane = lane;
  w.qf = reinterpret_cast<const uint4*>(frag) + lane;
  w.qsum = qsum;
  w.factor = factor;
  w.limit = limit;
  w.shift = reinterpret_cast<float*>(frag + C::QFRAG) + warp * C::NG * C::COLS;
  uint8_t* const ring = smem + warp * C::STAGES * C::STAGE;
  const uint32_t ring_at = smem_addr(ring);

  Item it{};
  constexpr int Q4 = C::D / 4;
  constexpr int PART = C::COLS * (C::D + 2);                       // floats of a partial result
  auto write = [&](int col, int d, float4 x, float sum) {          // a piece of a row of the result
    int h;
    const int i = by_group.of(it.row0 + col, h);
    const bool empty = i >= it.n || sum == 0.f;
    const float inv = empty ? 0.f : 1.f / sum;
    uint2 y = make_uint2(pack<T>(x.x * inv, x.y * inv), pack<T>(x.z * inv, x.w * inv));
    if (empty) y = make_uint2(0, 0);
    *reinterpret_cast<uint2*>((T*)p.out.p + it.seq * p.out.st.b + (it.head * p.group + h) * p.out.st.h + i * p.out.st.s + d) = y;
  };
  int i0 = 0, i1 = 0;                                              // CTAs that share the item
  while (unit < unit_end) {
    // the item of this unit
    int lo = 0, hi = bt.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (prefix[mid] <= unit) lo = mid;
      else hi = mid - 1;
    }
    it.seq = lo;
    it.full = bt.seq_lens[lo];
    it.len = max(0, min(it.full, table_tokens));
    const int units = max(1, (it.len + unit_tokens - 1) >> unit_shift);
    int start;
    const int within = unit - prefix[lo], index = Divisor(units).of(within, start);
    const int item_first = unit - start;
    it.unit1 = item_first + units;
    const int stop = min(unit_end, it.unit1);
    it.row0 = Divisor(c.kv_heads).of(index, it.head) * C::COLS;
    it.n = bt.new_lens ? min(max(bt.new_lens[lo], 0), bt.new_tokens) : bt.new_tokens;
    {
      const int i0 = by_group.of(it.row0), i1 = min(by_group.of(it.row0 + C::COLS - 1), it.n - 1);
      it.first = max(0, min(it.len, it.full - it.n + i0 + 1));
      it.end = i0 <= i1 ? max(0, min(it.len, it.full - it.n + i1 + 1)) : 0;
    }
    const int tok0 = start * unit_tokens, tok1 = min(it.end, (start + stop - unit) * unit_tokens);
    const int tiles = tok1 > tok0 ? (tok1 - tok0 + C::TILE - 1) / C::TILE : 0;
    const int mine = max(0, (tiles - warp + C::WARPS - 1) / C::WARPS);

    constexpr int ES = C::BITS == 16 ? 2 : 1;
    const uint8_t* const kb = (const uint8_t*)c.k + it.head * c.k_strides[1] * ES + lane % C::CH * 16;
    const uint8_t* const vb = (const uint8_t*)c.v + it.head * c.v_strides[1] * ES + lane % C::CH * 16;
    constexpr int PS = C::BITS == 8 ? 4 : 2;
    const uint8_t* const kpb = (const uint8_t*)c.k_params + PS * it.head * c.k_params_strides[1];
    const uint8_t* const vpb = (const uint8_t*)c.v_params + PS * it.head * c.v_params_strides[1];
    const int* const table = bt.block_table + it.seq * bt.table_stride;
    int page[C::MT];
    uint32_t holes = 0;                                            // 16 tokens without a page: bit (place in the ring) * MT + m
    int next = tok0 + warp * C::TILE;                              // first token of the tile whose pages are fetched next
    auto lookup = [&](int t) { return t < tok1 ? table[t >> p.a.shift] : -1; };
    auto fetch = [&](int (&page)[C::MT]) {                         // pages of the next tile, which issue() looks at, so that nothing waits for them here
      page[0] = lookup(next);
      if constexpr (C::MT == 2) page[1] = p.a.shift > 4 ? page[0] : lookup(next + 16);   // (tiles start at multiples of 32)
      next += C::UNIT;
    };
    auto issue = [&](int slot, int t0, const int (&fetched)[C::MT]) {        // the copies of a tile, to this place in the ring, once its pages are here
      const uint32_t at = ring_at + slot * C::STAGE;
      int page[C::MT];
#pragma unroll
      for (int m = 0; m < C::MT; ++m) {
        const bool there = (unsigned)fetched[m] < (unsigned)c.num_pages;
        if (!there && t0 + 16 * m < tok1) paged_fault(p.a, PBS_PAGED_BAD_PAGE);
        page[m] = there ? fetched[m] : -1;
      }
      if constexpr (C::BITS == 8) {                                // scales: a lane one
        const int m = lane >> 1, pg = C::MT == 2 && m == 1 ? page[C::MT - 1] : page[0], first = t0 + 16 * m;
        if (m < C::MT && pg >= 0 && first < tok1) {
          const uint32_t block = (first & (c.page_size - 1)) >> p.a.block_shift;
          copy_async<4>(at + 2 * C::TILE * C::ROW + 4 * lane,
                        lane & 1 ? vpb + 4 * (uint64_t)(pg * p.vp_page + block * p.vp_slot) : kpb + 4 * (uint64_t)(pg * p.kp_page + block * p.kp_slot));
        }
      }
      if (p.dense && t0 + C::TILE <= tok1 && page[0] >= 0 && page[C::MT - 1] >= 0) {
        // the common case, whose copies are a few constants away from one another: half the instructions of the one below
        holes &= ~(((1u << C::MT) - 1) << slot * C::MT);
#pragma unroll
        for (int m = 0; m < C::MT; ++m) {
          const uint32_t sl = (t0 + 16 * m) & (c.page_size - 1);
          const uint8_t* const ks = kb + 16 * (uint64_t)(page[m] * p.k_page + sl * (uint32_t)C::CH + lane / C::CH * C::CH);
          const uint8_t* const vs = vb + 16 * (uint64_t)(page[m] * p.v_page + sl * (uint32_t)C::CH + lane / C::CH * C::CH);
#pragma unroll
          for (int s = 0; s < C::CH / 2; ++s) {
            const int dst = piece<C>(16 * m + lane / C::CH + s * (32 / C::CH), lane % C::CH);
            copy_async<16>(at + dst, ks + s * 512);
            copy_async<16>(at + C::TILE * C::ROW + dst, vs + s * 512);
          }
        }
        if constexpr (C::BITS == 4) {
          constexpr int N = C::PROW < 16 ? C::PROW : 16;
          const int row = lane % C::TILE, pg = C::MT == 2 && row >= 16 ? page[C::MT - 1] : page[0];
          const uint32_t sl = (t0 + row) & (c.page_size - 1), dst = at + 2 * C::TILE * C::ROW + row * C::PROW;
          const uint8_t* const ks = kpb + 4 * (uint64_t)(pg * p.kp_page + sl * (uint32_t)C::NG);
          const uint8_t* const vs = vpb + 4 * (uint64_t)(pg * p.vp_page + sl * (uint32_t)C::NG);
#pragma unroll
          for (int o = 0; o < C::PROW; o += N) {
            if (C::TILE == 32 || lane < 16) copy_async<N>(dst + o, ks + o);
            if (C::TILE == 32 || lane >= 16) copy_async<N>(dst + C::TILE * C::PROW + o, vs + o);
          }
        }
        return;
      }
#pragma unroll
      for (int m = 0; m < C::MT; ++m) {
        const bool there = page[m] >= 0;
        const uint32_t hole = 1u << (slot * C::MT + m), pg = there ? page[m] : 0, sl = (t0 + 16 * m) & (c.page_size - 1);
        holes = there ? holes & ~hole : holes | hole;
        const int rows = there ? tok1 - t0 - 16 * m : 0;           // (offsets stay within the page also for those that are only filled)
        const uint32_t ko = pg * p.k_page + (sl + lane / C::CH) * p.k_slot, vo = pg * p.v_page + (sl + lane / C::CH) * p.v_slot;
#pragma unroll
        for (int s = 0; s < C::CH / 2; ++s) {
          const int row = lane / C::CH + s * (32 / C::CH), dst = piece<C>(16 * m + row, lane % C::CH);
          copy_async<16>(at + dst, kb + 16 * (uint64_t)(ko + s * (32 / C::CH) * p.k_slot), row < rows);
          copy_async<16>(at + C::TILE * C::ROW + dst, vb + 16 * (uint64_t)(vo + s * (32 / C::CH) * p.v_slot), row < rows);
        }
      }
      if constexpr (C::BITS == 4) {
        constexpr int N = C::PROW < 16 ? C::PROW : 16;
        const int row = lane % C::TILE, pgm = C::MT == 2 && row >= 16 ? page[C::MT - 1] : page[0];
        const bool copy = pgm >= 0 && t0 + row < tok1;
        const uint32_t pg = pgm >= 0 ? pgm : 0, sl = (t0 + row) & (c.page_size - 1), dst = at + 2 * C::TILE * C::ROW + row * C::PROW;
        const uint8_t* const ks = kpb + 4 * (uint64_t)(pg * p.kp_page + sl * p.kp_slot);
        const uint8_t* const vs = vpb + 4 * (uint64_t)(pg * p.vp_page + sl * p.vp_slot);
#pragma unroll
        for (int o = 0; o < C::PROW; o += N) {
          if (C::TILE == 32 || lane < 16) copy_async<N>(dst + o, ks + o, copy);
          if (C::TILE == 32 || lane >= 16) copy_async<N>(dst + C::TILE * C::PROW + o, vs + o, copy);
        }
      }
    };
    // the queries and the pages of the first tiles on their way together: one after the other they took 5 us under load
    Queries<C> queries;
    queries.load(p, it, by_group);
    int first_pages[C::STAGES - 1][C::MT];
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; ++s) fetch(first_pages[s]);
    fetch(page);
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; ++s) {
      if (s < mine) issue(s, tok0 + warp * C::TILE + s * C::UNIT, first_pages[s]);
      copy_commit();
    }
    queries.put(p, it, by_group, frag, qsum, factor, limit);
    w.start();
    __syncthreads();
    int slot = 0, t0 = tok0 + warp * C::TILE;
    const int plain = min(it.first, tok1) - C::TILE;               // tiles up to here are seen whole by all queries
    for (int i = 0; i < mine; ++i, t0 += C::UNIT) {
      copy_wait<C::STAGES - 2>();
      __syncwarp();                                                // (the place read last is free in all lanes, too)
      if (i + C::STAGES - 1 < mine) issue(slot == 0 ? C::STAGES - 1 : slot - 1, t0 + (C::STAGES - 1) * C::UNIT, page);
      fetch(page);
      copy_commit();
      const uint8_t* stage = ring + slot * C::STAGE;
      const uint32_t hole = holes >> slot * C::MT & ((1u << C::MT) - 1);
      if (t0 > plain || hole) w.template tile<true>(stage, t0, hole);
      else w.template tile<false>(stage, t0, 0);
      if ((C::SHIFT > 0 || C::BITS == 8) && i % kShiftEvery == kShiftEvery - 1) w.move_sums();
      slot = slot == C::STAGES - 1 ? 0 : slot + 1;
    }
    copy_wait<0>();
    __syncthreads();                                               // the ring is free: partial sums take its place
    float* sums = reinterpret_cast<float*>(smem);
    float* refs = sums + C::WARPS * C::COLS * C::OROW;
    float* weights = refs + C::WARPS * C::COLS;
    w.put(sums + warp * C::COLS * C::OROW, refs + warp * C::COLS, weights + warp * C::COLS);
    __syncthreads();

    i0 = by_share.of(item_first);
    i1 = by_share.of(it.unit1 - 1);
    const int cols = min(C::COLS, bt.new_tokens * p.group - it.row0);
    float* const part = p.partials + ((int64_t)blockIdx.x * 2 + ((int)blockIdx.x == i0)) * PART;
    for (int e = tid; e < cols * Q4; e += C::THREADS) {
      const int col = e / Q4, d = e % Q4 * 4;
      float top = -CUDART_INF_F, sum = 0.f;
#pragma unroll
      for (int v = 0; v < C::WARPS; ++v) top = fmaxf(top, refs[v * C::COLS + col]);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int v = 0; v < C::WARPS; ++v) {
        const float rv = refs[v * C::COLS + col], wt = rv == top ? 1.f : factor_of<C>(rv - top);
        const float4 y = *reinterpret_cast<const float4*>(sums + (v * C::COLS + col) * C::OROW + d);
        sum = add_scaled<C>(wt, weights[v * C::COLS + col], sum);
        x.x = add_scaled<C>(wt, y.x, x.x);
        x.y = add_scaled<C>(wt, y.y, x.y);
        x.z = add_scaled<C>(wt, y.z, x.z);
        x.w = add_scaled<C>(wt, y.w, x.w);
      }
      if (i0 == i1) {
        write(col, d, x, sum);
      } else {
        __stcg(reinterpret_cast<float4*>(part + col * C::D + d), x);
        if (d == 0) {
          __stcg(part + C::COLS * C::D + col, top);
          __stcg(part + C::COLS * (C::D + 1) + col, sum);
        }
      }
    }
    __syncthreads();
    if (i0 != i1 && tid == 0 && !(p.drop_arrive && blockIdx.x == 0)) {
      __threadfence();                                             // (after the barrier above: for the whole CTA's stores)
      atomicAdd(p.counters + 2 * i0, 1u);
    }
    unit = stop;
  }
  if (i0 == i1) return;

  // The CTAs whose last item this is (the one behind its end may have gone on to another) wait for all parts and join a share of the pieces each
  const int n = i1 - i0 + 1, joiners = min(total, (i1 + 1) * share) > it.unit1 ? n - 1 : n;
  if (tid == 0) {
    volatile unsigned* const parts = p.counters + 2 * i0;
    unsigned long long start, now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
    do {
      arrived = *parts == (unsigned)n;
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    } while (!arrived && now - start < p.wait_ns);
    __threadfence();
    if (!arrived) {
      paged_fault(p.a, PBS_PAGED_TIMEOUT);
    } else if (atomicAdd(p.counters + 2 * i0 + 1, 1u) == (unsigned)joiners - 1) {        // all have seen it: for the next call
      p.counters[2 * i0] = 0;
      p.counters[2 * i0 + 1] = 0;
    }
  }
  __syncthreads();
  if (!arrived) return;
  const int pieces = min(C::COLS, bt.new_tokens * p.group - it.row0) * Q4, per_cta = (pieces + joiners - 1) / joiners;
  const int e0 = ((int)blockIdx.x - i0) * per_cta, e1 = min(pieces, e0 + per_cta);
  auto from = [&](int k) { return p.partials + ((int64_t)(i0 + k) * 2 + (k == 0)) * PART; };
  if (n <= 8) {                                                    // few parts: a thread a piece
    for (int e = e0 + tid; e < e1; e += C::THREADS) {
      const int col = e / Q4, d = e % Q4 * 4;
      float top = -CUDART_INF_F, sum = 0.f, rv[8], lv[8];
      float4 y[8], x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        rv[k] = -CUDART_INF_F;
        lv[k] = 0.f;
        y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k >= n) continue;
        rv[k] = __ldcg(from(k) + C::COLS * C::D + col);
        lv[k] = __ldcg(from(k) + C::COLS * (C::D + 1) + col);
        y[k] = __ldcg(reinterpret_cast<const float4*>(from(k) + col * C::D + d));
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, rv[k]);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float wt = rv[k] == top ? 1.f : factor_of<C>(rv[k] - top);
        sum = add_scaled<C>(wt, lv[k], sum);
        x.x = add_scaled<C>(wt, y[k].x, x.x);
        x.y = add_scaled<C>(wt, y[k].y, x.y);
        x.z = add_scaled<C>(wt, y[k].z, x.z);
        x.w = add_scaled<C>(wt, y[k].w, x.w);
      }
      write(col, d, x, sum);
    }
    return;
  }
  for (int e = e0 + warp; e < e1; e += C::WARPS) {                 // many: a warp a piece
    const int col = e / Q4, d = e % Q4 * 4;
    float top = -CUDART_INF_F, sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = lane; k0 - lane < n; k0 += 128) {
      float rv[4], lv[4];
      float4 y[4];
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        rv[a] = -CUDART_INF_F;
        lv[a] = 0.f;
        y[a] = make_float4(0.f, 0.f, 0.f, 0.f);
        const int k = k0 + 32 * a;
        if (k >= n) continue;
        rv[a] = __ldcg(from(k) + C::COLS * C::D + col);
        lv[a] = __ldcg(from(k) + C::COLS * (C::D + 1) + col);
        y[a] = __ldcg(reinterpret_cast<const float4*>(from(k) + col * C::D + d));
      }
      const float most = fmaxf(top, warp_max(fmaxf(fmaxf(rv[0], rv[1]), fmaxf(rv[2], rv[3])))), keep = top == most ? 1.f : factor_of<C>(top - most);
      top = most;
      sum = scaled<C>(sum, keep);
      x = make_float4(scaled<C>(x.x, keep), scaled<C>(x.y, keep), scaled<C>(x.z, keep), scaled<C>(x.w, keep));
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const float wt = rv[a] == top ? 1.f : factor_of<C>(rv[a] - top);
        sum = add_scaled<C>(wt, lv[a], sum);
        x.x = add_scaled<C>(wt, y[a].x, x.x);
        x.y = add_scaled<C>(wt, y[a].y, x.y);
        x.z = add_scaled<C>(wt, y[a].z, x.z);
        x.w = add_scaled<C>(wt, y[a].w, x.w);
      }
    }
    x = make_float4(warp_sum(x.x), warp_sum(x.y), warp_sum(x.z), warp_sum(x.w));
    sum = warp_sum(sum);
    if (lane == 0) write(col, d, x, sum);
  }
}

// Shared memory of a SM, and what a CTA takes of it beyond its dynamic part.
constexpr int kSmemPerSm = 228 * 1024, kOverhead = 1024 + 256;

// NT: the narrowest that holds all queries of a KV head, or the widest (of 256 channels two, for its registers).  Columns that hold no query
// cost as much as others: 20 queries over pages of 16 bits (8 sequences of up to 8192) take 39.7 us in three, 41.7 in four.
int query_tiles(const PagedArgs& a, int q_heads) {
  const int64_t rows = (int64_t)q_heads / a.c.kv_heads * a.b.new_tokens;
  return rows <= 8 ? 1 : rows <= 16 || a.c.head_dim == 256 ? 2 : rows <= 24 ? 3 : 4;
}

template <class C>
int launch(AttnArgs p, void* workspace, bool measure, int64_t* bytes, cudaStream_t st) {
  const int64_t rows = (int64_t)p.group * p.a.b.new_tokens;
  p.row_tiles = (int)((rows + C::COLS - 1) / C::COLS);
  const int64_t most = ((int64_t)p.a.b.max_pages * p.a.c.page_size / C::UNIT + 1) * p.row_tiles * p.a.c.kv_heads * p.a.b.batch;
  if (most > INT_MAX - (1 << 20)) { set_error("paged attention: sequences x heads x tokens beyond what a call can count"); return PBS_ERR_SHAPE; }
  // One CTA a SM where that leaves at most kShort units each (by the table, whose sequences may be shorter): what a second one saves on a
  // few tiles goes on joining twice the parts.  One sequence of 32768 with 4 KV heads 13.6 us so, 14.7 with two; of 131072 with 8, 28
  // units each, 47.4 against 44.5.
  constexpr int kShort = 8;
  const int sms = device_sms();
  int grid = most <= (int64_t)kShort * sms ? sms : C::OCC * sms;
  const int bytes_smem = C::FIXED + p.a.b.batch * 4;
  if (2 * (bytes_smem + kOverhead) > kSmemPerSm && grid > sms) grid = sms;     // (all CTAs have to be resident)
  if (grid > kMaxGrid) grid = kMaxGrid;
  if (most < grid) grid = (int)most;
  if (measure) {
    *bytes = PBS_PAGED_COUNTER_BYTES + (int64_t)grid * 2 * C::COLS * (C::D + 2) * 4;
    return PBS_OK;
  }
  const pbs_paged_cache_t& c = p.a.c;
  bool fits = true;
  auto steps = [&](const int64_t (&st)[3], int bytes, int unit, uint32_t& page, uint32_t& slot, int rows) {
    const int64_t a = st[0] * bytes / unit, b = st[2] * bytes / unit;
    fits = fits && a <= UINT32_MAX && b <= UINT32_MAX && (__int128)(c.num_pages - 1) * a + (__int128)(rows - 1) * b <= UINT32_MAX;
    page = (uint32_t)a;
    slot = (uint32_t)b;
  };
  p.dense = c.k_strides[2] * (C::BITS == 16 ? 2 : 1) == C::ROW && c.v_strides[2] * (C::BITS == 16 ? 2 : 1) == C::ROW &&
            (C::BITS != 4 || (c.k_params_strides[2] == 2 * C::NG && c.v_params_strides[2] == 2 * C::NG));
  steps(c.k_strides, C::BITS == 16 ? 2 : 1, 16, p.k_page, p.k_slot, c.page_size);
  steps(c.v_strides, C::BITS == 16 ? 2 : 1, 16, p.v_page, p.v_slot, c.page_size);
  if (C::BITS != 16) {
    const int rows = C::BITS == 4 ? c.page_size : c.page_size >> p.a.block_shift;
    steps(c.k_params_strides, C::BITS == 4 ? 2 : 4, 4, p.kp_page, p.kp_slot, rows);
    steps(c.v_params_strides, C::BITS == 4 ? 2 : 4, 4, p.vp_page, p.vp_slot, rows);
  }
  if (!fits) { set_error("paged attention: a pool of more than 64 GiB (params: 16 GiB)"); return PBS_ERR_SHAPE; }
  p.counters = (unsigned*)workspace;
  // an item may be long enough for several CTAs
  const bool splits = (int64_t)p.a.b.max_pages * p.a.c.page_size > (C::BITS == 8 ? kWhole : 1) * C::UNIT;
  p.wait_ns = g_wait_ns.load(std::memory_order_relaxed);
  p.drop_arrive = g_drop_arrive.load(std::memory_order_relaxed);
  p.partials = (float*)((uint8_t*)workspace + PBS_PAGED_COUNTER_BYTES);
  // the limit that holds for any batch, set once a device
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !(allowed.load(std::memory_order_relaxed) >> dev & 1))) {
    e = cudaFuncSetAttribute(paged_attn_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::FIXED + kMaxBatch * 4);
    if (e == cudaSuccess && dev < 64) allowed.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return cuda_fail(e, "paged_attn_kernel shared memory");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = bytes_smem;
  cfg.stream = st;
  cudaLaunchAttribute together = {};
  together.id = cudaLaunchAttributeCooperative;
  together.val.cooperative = 1;
  cudaLaunchAttribute early = early_launch();
  cfg.attrs = splits ? &together : &early;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, paged_attn_kernel<C>, p);
  if (e != cudaSuccess) return cuda_fail(e, "paged_attn_kernel");
  PBS_CUDA_CHECK_LAUNCH("paged_attn_kernel");
  return PBS_OK;
}

template <int DT, int D, int BITS, int G>
int by_queries(const AttnArgs& p, void* w, bool measure, int64_t* bytes, cudaStream_t st) {
  const int nt = query_tiles(p.a, p.q_heads);
  if (nt == 1) return launch<Cfg<DT, D, BITS, G, 1>>(p, w, measure, bytes, st);
  if constexpr (D != 256)
    if (nt == 3) return launch<Cfg<DT, D, BITS, G, 3>>(p, w, measure, bytes, st);
  if constexpr (D != 256)
    if (nt == 4) return launch<Cfg<DT, D, BITS, G, 4>>(p, w, measure, bytes, st);
  return launch<Cfg<DT, D, BITS, G, 2>>(p, w, measure, bytes, st);
}

template <int DT, int D>
int by_bits(const AttnArgs& p, void* w, bool measure, int64_t* bytes, cudaStream_t st) {
  if (p.a.c.bits == 16) return by_queries<DT, D, 16, D>(p, w, measure, bytes, st);
  if (p.a.c.bits == 8) return by_queries<DT, D, 8, D>(p, w, measure, bytes, st);
  return p.a.c.group_size == 32 ? by_queries<DT, D, 4, 32>(p, w, measure, bytes, st) : by_queries<DT, D, 4, 64>(p, w, measure, bytes, st);
}

template <int DT>
int by_dim(const AttnArgs& p, void* w, bool measure, int64_t* bytes, cudaStream_t st) {
  return p.a.c.head_dim == 64 ? by_bits<DT, 64>(p, w, measure, bytes, st)
         : p.a.c.head_dim == 128 ? by_bits<DT, 128>(p, w, measure, bytes, st) : by_bits<DT, 256>(p, w, measure, bytes, st);
}

int by_type(const AttnArgs& p, void* w, bool measure, int64_t* bytes, cudaStream_t st) {
  return p.a.c.dtype == PBS_BF16 ? by_dim<PBS_BF16>(p, w, measure, bytes, st) : by_dim<PBS_FP16>(p, w, measure, bytes, st);
}

}  // namespace

int paged_attn_workspace(const PagedArgs& a, int q_heads, int64_t* bytes) {
  AttnArgs p{};
  p.a = a;
  p.q_heads = q_heads;
  p.group = q_heads / a.c.kv_heads;
  return by_type(p, nullptr, true, bytes, nullptr);
}

int launch_paged_attn(const PagedArgs& a, int q_heads, const RowTensor& q, const RowTensor& out, float scale, void* workspace, cudaStream_t st) {
  AttnArgs p{};
  p.a = a;
  p.q = q;
  p.out = out;
  p.q_heads = q_heads;
  p.group = q_heads / a.c.kv_heads;
  p.scale = scale * 1.44269504f;
  return by_type(p, workspace, false, nullptr, st);
}

void set_paged_wait(unsigned long long wait_ns, int drop_arrive) {
  g_wait_ns.store(wait_ns ? wait_ns : 2000000000ull, std::memory_order_relaxed);
  g_drop_arrive.store(drop_arrive, std::memory_order_relaxed);
}

}  // namespace pbs
