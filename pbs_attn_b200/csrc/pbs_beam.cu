// The best continuations of each batch entry's beams: log-softmax of every beam's logits, plus its score, and the K largest of all beams and tokens.
//
// Within a beam the order of the scores is the order of the logits, so one pass over the logits gives both what the softmax needs (their maximum and
// the sum of exponentials) and each slice's K largest; scores are formed for these few only, in 64 bits, when a batch entry's slices meet.
//
// A CTA takes a segment of a row, in chunks of two 16-byte pieces a thread; the chunks ahead are on their way to shared memory meanwhile (each
// thread's own pieces: nobody waits for anybody).  A thread keeps its sum, and the largest logits of its three best chunks.  At the end the
// threads' largest give a bound that K logits reach, and few more: the chunks that do are looked at once more, their logits listed and ranked by
// counting.  Order: (logit, then lower token) as one 64-bit number, so that ties need no case of their own.  (With lists kept while streaming,
// cut down to K now and then, the CTA's warps waited for one another and branched: 76 us for 512 rows of 152064 in fp32.)
// The CTA that finishes an entry last merges the sorted lists of its segments in the same way, by score.
//
// Measured (B200, GPU time): 512 rows of 152064 in fp32, 64 entries of eight beams, 61 to 64 us, 74 to 78 % of the copy rate: streaming runs at it, the
// segments' ends and the merges (5 us each) behind it do not overlap much, as all rows end at once; in bf16 50 us, 47 %: 23 us of instruction issue
// and 20 of exponentials, which come one after the other in every warp.  64 rows of 128256 in bf16 17 us, four 11, one 10: latency of 20000 cycles, of
// which the meeting of the segments (fence, count, loads, ranks) is more than half.
#include <climits>

#include "pbs_paged.cuh"

namespace pbs {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int P = 2, kStages = 3;          // 16-byte pieces of a thread in a chunk; chunks in shared memory, all but one of them on their way
constexpr int kResident = 4;              // CTAs a SM
constexpr int kListed = 1024;             // logits that reach the bound; of more the K-th of those that found room is a better bound
constexpr int kSample = 512;              // of these
constexpr int kFound = 320;               // continuations that do
constexpr int kMaxBeams = 32;
constexpr float kFltMax = 3.402823466e38f;
constexpr float kLog2e = 1.44269504f;

struct BeamArgs {
  pbs_beam_select_t a;
  int slices, chunks, share;              // segments of a row; chunks of a row, and of a segment
  unsigned* counters;                     // by batch entry: segments that are done
  float2* sums;                           // by segment: maximum, sum of exponentials
  unsigned long long* lists;              // by segment: its K largest
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\nfma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// A number whose order is that of (value, then lower token); 0 is none.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);             // (-0 is 0)
  return b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key ^ ((int)key < 0 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ unsigned long long ordered(float x, int token) { return (unsigned long long)key_of(x) << 32 | ~(uint32_t)token; }
__device__ __forceinline__ unsigned long long key_of(double x) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(x + 0.0);
  return b ^ ((long long)b < 0 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double value_of(unsigned long long key) {
  return __longlong_as_double((long long)(key ^ ((long long)key < 0 ? 1ull << 63 : ~0ull)));
}

// The elements of a 16-byte piece, as floats and back.
template <class T>
struct Piece;
template <>
struct Piece<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& w, float (&x)[4]) {
    x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ uint4 put(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ float most(const uint4& w) {
    return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
};
template <>
struct Piece<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 put(const float (&x)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(x[2 * i]) >> 16 | (__float_as_uint(x[2 * i + 1]) & 0xffff0000u);
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ float most(const uint4& w) {
    const __nv_bfloat162 m = __hmax2(__hmax2(pair(w.x), pair(w.y)), __hmax2(pair(w.z), pair(w.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ __nv_bfloat162 pair(const uint32_t& u) { return *reinterpret_cast<const __nv_bfloat162*>(&u); }
};
template <>
struct Piece<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint4 put(const float (&x)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
  static __device__ __forceinline__ float most(const uint4& w) {
    const __half2 m = __hmax2(__hmax2(pair(w.x), pair(w.y)), __hmax2(pair(w.z), pair(w.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ __half2 pair(const uint32_t& u) { return *reinterpret_cast<const __half2*>(&u); }
};

// What a logit counts as.
__device__ __forceinline__ float counted(float x) { return x == x ? x : -CUDART_INF_F; }

// A number that K of the CTA's (one a thread) reach, and few more where warps' numbers are alike: what ceil(K / warps) of every warp do.
// (Short, and not inlined: in a kernel of this size code that is not there yet takes longer than what it does.  The exact K-th largest, by the places of
// the warps' sorted numbers among all, took 3000 cycles more.)
__device__ __noinline__ float bound_of(float x, int K, float* meet) {
  uint32_t left = key_of(x), top = 0;
  for (int i = (K - 1) / kWarps; i >= 0; --i) {            // (equal ones go one by one, so that K are K)
    top = __reduce_max_sync(0xffffffffu, left);
    if ((int)(threadIdx.x % 32) == __ffs(__ballot_sync(0xffffffffu, left == top)) - 1) left = 0;
  }
  if (threadIdx.x % 32 == 0) meet[threadIdx.x / 32] = value_of(top);
  __syncthreads();
  float least = meet[0];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) least = fminf(least, meet[i]);
  return least;
}

// The same where they may differ: what K of one warp reach, or of two for K above 32.  meet: not that of the other.
__device__ __noinline__ float bound_of_one(float x, int K, float* meet) {
  const int lane = threadIdx.x % 32;
#pragma unroll 1
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll 1
    for (int j = k >> 1; j > 0; j >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, x, j);
      x = ((lane & j) == 0) == ((lane & k) == 0 || k == 32) ? fmaxf(x, y) : fminf(x, y);
    }
  const float kth = __shfl_sync(0xffffffffu, x, min(K, 32) - 1);
  if (lane == 0) meet[threadIdx.x / 32] = kth;
  __syncthreads();
  float most = -CUDART_INF_F;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) most = fmaxf(most, K <= 32 ? meet[i] : fminf(meet[i], meet[i ^ 1]));
  return most;
}

// A continuation: its score's order, its beam, and its place in the beam (logit and token).
struct Next {
  unsigned long long score, place;        // 0: none
  uint32_t beam;
};
__device__ __forceinline__ bool before(const Next& a, const Next& b) {
  return a.score != b.score ? a.score > b.score : a.beam != b.beam ? a.beam < b.beam : a.place > b.place;
}

// Lane that holds the first of the warp's in the order of before().
__device__ __forceinline__ int first_lane(const Next& x) {
  uint32_t among = 0xffffffffu;
  auto keep = [&](uint32_t v) {                            // the lanes among them whose v is largest
    const bool in = among >> (threadIdx.x & 31) & 1;
    const uint32_t top = __reduce_max_sync(0xffffffffu, in ? v : 0u);
    among &= __ballot_sync(0xffffffffu, in && v == top);
    return (among & (among - 1)) == 0;
  };
  if (keep((uint32_t)(x.score >> 32)) || keep((uint32_t)x.score) || keep(~x.beam) || keep((uint32_t)(x.place >> 32)) || keep((uint32_t)x.place)) {}
  return __ffs(among) - 1;
}

// A row of logits.  Pieces are cut where addresses are multiples of 16.
template <class T>
struct Row {
  static constexpr int N = Piece<T>::N, CHUNK = kThreads * P * N;
  const T* in;
  int vocab, lead;                        // elements between a boundary and the row's first
  bool alive;                             // (a beam that is not has no order but the tokens')

  __device__ __forceinline__ Row(const pbs_beam_select_t& a, int row)
      : in((const T*)a.logits + row * a.logits_stride), vocab(a.vocab), lead((int)(((uintptr_t)in & 15) / sizeof(T))), alive(true) {}
  __device__ __forceinline__ bool has(int v) const { return (unsigned)v < (unsigned)vocab; }
  __device__ __forceinline__ float one(int v) const { return alive ? counted(Piece<T>::one(in + v)) : -CUDART_INF_F; }
  // Token of element i of a thread's piece k of a chunk, the first and last whole pieces, and whether a chunk has no others.
  __device__ __forceinline__ int token(int chunk, int k, int i, int thread) const { return chunk * CHUNK - lead + (k * kThreads + thread) * N + i; }
  __device__ __forceinline__ int token(int chunk, int k, int i) const { return token(chunk, k, i, (int)threadIdx.x); }
  __device__ __forceinline__ int whole0() const { return lead ? N - lead : 0; }
  __device__ __forceinline__ int whole1() const { return (vocab + lead) / N * N - lead - N; }
  __device__ __forceinline__ bool inner(int chunk) const { return chunk * CHUNK - lead >= whole0() && (chunk + 1) * CHUNK - lead - N <= whole1(); }

  // Copies of this thread's pieces, or, of those that are an end of the row or beyond it, of some other; ends() puts those right.
  __device__ __forceinline__ void copy(int chunk, uint4* to) const {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
    const bool plain = inner(chunk);
    if (plain) {
      const T* const from = in + token(chunk, 0, 0);
#pragma unroll
      for (int k = 0; k < P; ++k) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + k * kThreads * 16), "l"(from + k * kThreads * N) : "memory");
      return;
    }
    const int w0 = whole0(), w1 = whole1();
    if (w1 < w0) return;
#pragma unroll
    for (int k = 0; k < P; ++k)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + k * kThreads * 16), "l"(in + min(max(token(chunk, k, 0), w0), w1)) : "memory");
  }
  __device__ __forceinline__ void ends(int chunk, uint4 (&w)[P], int thread, bool all = false) const {
#pragma unroll
    for (int k = 0; k < P; ++k) {
      const int v = token(chunk, k, 0, thread);
      if (!all && alive && v >= whole0() && v <= whole1()) continue;
      float x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = alive && has(v + i) ? Piece<T>::one(in + v + i) : -CUDART_INF_F;
      w[k] = Piece<T>::put(x);
    }
  }
};

// A thread's logits so far: their maximum, and the sum of exp(logit - maximum).
struct Sum {
  float top = -kFltMax, sum = 0.f;

  // Takes in P pieces and returns the largest of their logits (a NaN counts as -infinity).
  template <class T>
  __device__ __forceinline__ float add(const uint4 (&w)[P]) {
    using E = Piece<T>;
    constexpr int N = E::N;
    float most = E::most(w[0]);
#pragma unroll
    for (int k = 1; k < P; ++k) most = fmaxf(most, E::most(w[k]));       // (a NaN gives way)
    if (!(most >= -kFltMax)) most = -CUDART_INF_F;
    const float higher = fmaxf(top, fminf(most, kFltMax)), shift = -higher * kLog2e;
    const float2 scale = make_float2(kLog2e, kLog2e), by = make_float2(shift, shift);
    float2 both = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < P; ++k) {
      float x[N];
      E::get(w[k], x);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float2 y = fma2(make_float2(x[i], x[i + 1]), scale, by);
        both = add2(both, make_float2(exp2_fast(y.x), exp2_fast(y.y)));
      }
    }
    float more = both.x + both.y;
    more *= exp2_fast(-fmaf(higher, kLog2e, shift));       // (what the rounding of the shift has made of them all)
    // Where logits are so large that this rounding matters, and where any is not a number or infinite: +infinity counts as the largest number.
    if (__any_sync(0xffffffffu, !(more <= kFltMax) || fabsf(higher) > 1e5f)) {
      more = 0.f;
#pragma unroll
      for (int k = 0; k < P; ++k) {
        float x[N];
        E::get(w[k], x);
#pragma unroll
        for (int i = 0; i < N; ++i) more += exp2_fast((fminf(counted(x[i]), kFltMax) - higher) * kLog2e);
      }
    }
    sum = sum * exp2_fast((top - higher) * kLog2e) + more;
    top = higher;
    return most;
  }
};

template <class T>
__global__ void __launch_bounds__(kThreads, kResident) beam_select_kernel(const __grid_constant__ BeamArgs p) {
  using E = Piece<T>;
  using R = Row<T>;
  constexpr int N = E::N;
  __shared__ __align__(16) uint4 ring[kStages][P][kThreads];
  __shared__ unsigned long long list[kListed];
  __shared__ unsigned long long found_score[kFound], found_place[kFound];
  __shared__ uint32_t found_beam[kFound];
  __shared__ Next heads[kWarps];
  __shared__ float2 part[kWarps];
  __shared__ float bounds[kWarps], bounds_of_one[kWarps];
  __shared__ unsigned long long kth;
  __shared__ int listed, last;
  __shared__ double norm[kMaxBeams];                       // of a beam: its score, less the logarithm of its sum
  __shared__ float peak[kMaxBeams];
  after_the_kernel_before();
  const pbs_beam_select_t& a = p.a;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, K = a.keep;
  const int r = blockIdx.x / p.slices, entry = r / a.beams;
  {
    const int chunk0 = (int)(blockIdx.x - r * p.slices) * p.share, chunk1 = min(p.chunks, chunk0 + p.share);
    R row(a, r);
    int ahead = chunk0, slot = 0;
    auto issue = [&] {
      if (ahead < chunk1) row.copy(ahead, &ring[(ahead - chunk0) % kStages][0][tid]);
      ++ahead;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue();
    row.alive = a.scores[entry * a.scores_stride + r % a.beams] > -CUDART_INF_F;
    if (tid == 0) listed = 0;
    Sum sum;
    float best[3] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};         // of this thread's chunks, and where the first two are
    int where[2] = {-1, -1};
    // (the logits of a beam that is not alive do not matter: 512 rows of 152064 in fp32, seven of eight so, as in a first step, 42 us against 65 of a later one)
    for (int c = chunk0; c < chunk1 && row.alive; ++c) {
      uint4 w[P];
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
#pragma unroll
      for (int k = 0; k < P; ++k) w[k] = ring[slot][k][tid];
      slot = (slot + 1) % kStages;
      issue();                                             // (into the place that was read before)
      if (!__all_sync(0xffffffffu, row.inner(c))) row.ends(c, w, tid);
      const float most = sum.add<T>(w);
      const bool first = most > best[0], second = most > best[1];
      best[2] = second ? best[1] : fmaxf(best[2], most);
      best[1] = first ? best[0] : second ? most : best[1];
      where[1] = first ? where[0] : second ? c : where[1];
      best[0] = first ? most : best[0];
      where[0] = first ? c : where[0];
    }
    // K logits reach the bound.  Where there are no K to reach anything, all that is not -infinity does, and the first K tokens of the segment,
    // enough of which are -infinity to fill up.
    float bound = -CUDART_INF_F;
    if (row.alive) {
      bound = bound_of(best[0], K, bounds);
      if (bound == -CUDART_INF_F) bound = bound_of_one(best[0], K, bounds_of_one);          // (a segment of few tokens, or most of them banned)
    } else {
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncthreads();                                     // (for `listed`, as in bound_of)
    }
    int filled = bound == -CUDART_INF_F ? max(chunk0 * R::CHUNK - row.lead, 0) + K : -1;
    int tie = INT_MAX;                                     // tokens up to this one reach the bound by being equal to it
    auto enlist = [&](int c, int thread) {                 // a thread's pieces of a chunk
      const bool plain = row.alive && row.inner(c);
      uint4 w[P];
#pragma unroll
      for (int k = 0; k < P; ++k) w[k] = plain ? __ldcg(reinterpret_cast<const uint4*>(row.in + row.token(c, k, 0, thread))) : make_uint4(0, 0, 0, 0);
      if (!plain) row.ends(c, w, thread, true);
      uint32_t reach = 0;
#pragma unroll
      for (int k = 0; k < P; ++k) {
        float x[N];
        E::get(w[k], x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int v = row.token(c, k, i, thread);
          if ((x[i] >= bound && x[i] > -CUDART_INF_F && (v <= tie || x[i] > bound)) || (v < filled && c == chunk0)) reach |= row.has(v) ? 1u << (k * N + i) : 0;
        }
      }
      for (; reach; reach &= reach - 1) {
        const int bit = __ffs(reach) - 1, v = row.token(c, bit / N, bit % N, thread);
        const int n = atomicAdd(&listed, 1);
        if (n >= kListed) break;
        list[n] = ordered(row.one(v), v);
      }
    };
    // (in three or more chunks of a thread: rarely, and then the warp looks through all of them)
    const uint32_t everywhere = __ballot_sync(0xffffffffu, best[2] >= bound && best[2] > -CUDART_INF_F);
    for (uint32_t left = everywhere; left; left &= left - 1)
      for (int c = chunk0 + lane; c < chunk1 && *(volatile int*)&listed <= kListed; c += 32) enlist(c, warp * 32 + __ffs(left) - 1);
    if (!(everywhere >> lane & 1)) {
      const bool fills = row.token(chunk0, 0, 0) < filled;
      if (fills) enlist(chunk0, tid);
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        const int c = i == 0 ? where[0] : where[1];
        if ((i == 0 ? best[0] : best[1]) >= bound && c >= 0 && !(fills && c == chunk0)) enlist(c, tid);
      }
    }
    // the segment's maximum and sum, and its list
    const float wide = warp_max(sum.top), scaled = warp_sum(sum.sum * exp2_fast((sum.top - wide) * kLog2e));
    if (lane == 0) part[warp] = make_float2(wide, scaled);
    __syncthreads();
    // Too many (equal ones, as where a mask is of the lowest finite number, or large ones in few threads' hands): the K-th of some that found room is a
    // better bound, which so many fewer reach, and of a sample of them a small part.  (512 rows of 152064 with five tokens that are not banned: 274 us,
    // four to five times as long as usual; gone through once for each of K = 16, as it was, 2820.)
    while (listed > kListed) {
      for (int i = tid; i < kSample; i += kThreads) {
        const unsigned long long mine = list[i];
        int at = 0;
#pragma unroll 4
        for (int j = 0; j < kSample; ++j) at += list[j] > mine;
        if (at == K - 1) kth = mine;
      }
      __syncthreads();
      bound = value_of((uint32_t)(kth >> 32));
      tie = (int)~(uint32_t)kth;
      filled = -1;                                         // (more than K are not -infinity)
      if (tid == 0) listed = 0;
      __syncthreads();
      for (int c = chunk0; c < chunk1; ++c) enlist(c, tid);
      __syncthreads();
    }
    const int n = listed;
    unsigned long long* const out = p.lists + (int64_t)blockIdx.x * K;
    for (int i = tid; i < n; i += kThreads) {
      const unsigned long long mine = list[i];
      int at = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) at += list[j] > mine;
      if (at < K) out[at] = mine;
    }
    for (int i = n + tid; i < K; i += kThreads) out[i] = 0;                // (a segment of fewer tokens)
    if (warp == 1) {
      const float2 x = lane < kWarps ? part[lane] : make_float2(-kFltMax, 0.f);
      const float m = warp_max(x.x), total = warp_sum(x.y * exp2_fast((x.x - m) * kLog2e));
      if (lane == 0) p.sums[blockIdx.x] = make_float2(m, total);
    }
  }
  __syncthreads();
  if (tid == 0) {
    __threadfence();                                       // (after the barrier: for the whole CTA's stores)
    last = atomicAdd(p.counters + entry, 1u) == (unsigned)(a.beams * p.slices) - 1;
    if (last) {
      p.counters[entry] = 0;                               // for the next call
      __threadfence();
    }
    listed = 0;
  }
  __syncthreads();
  if (!last) return;

  // The entry's segments meet.  A thread looks through a segment's sorted list, or several, or every g-th place of one where they are few.
  const int rows = a.beams, lists = rows * p.slices, number0 = entry * lists;
  const int g = lists >= kThreads ? 1 : min(K, kThreads / lists), together = kThreads / g;      // threads of a list; lists at a time
  const int list0 = tid / g < together ? tid / g : lists, place0 = tid % g;
  auto place_of = [&](int l, int i) { return __ldcg(p.lists + (int64_t)(number0 + l) * K + i); };
  const unsigned long long early = list0 < lists ? place_of(list0, place0) : 0;          // (on its way while the sums are added up)
  const int share = rows < kWarps ? kWarps / rows : 1;   // warps of a row, which all do the same
  constexpr int A = 4;                                   // loads under way
  for (int i = warp / share; i < rows; i += kWarps / share) {
    const float2* const sums = p.sums + number0 + i * p.slices;
    float2 x[A];
#pragma unroll
    for (int u = 0; u < A; ++u) x[u] = lane + u * 32 < p.slices ? __ldcg(sums + lane + u * 32) : make_float2(-kFltMax, 0.f);
    float m = -kFltMax, total = 0.f;
#pragma unroll 1
    for (int at = lane;;) {
      float wide = m;
#pragma unroll
      for (int u = 0; u < A; ++u) wide = fmaxf(wide, x[u].x);
      total *= exp2_fast((m - wide) * kLog2e);
#pragma unroll
      for (int u = 0; u < A; ++u) total += x[u].y * exp2_fast((x[u].x - wide) * kLog2e);
      m = wide;
      at += A * 32;
      if (at - lane >= p.slices) break;
#pragma unroll
      for (int u = 0; u < A; ++u) x[u] = at + u * 32 < p.slices ? __ldcg(sums + at + u * 32) : make_float2(-kFltMax, 0.f);
    }
    const float top = warp_max(m);
    total = warp_sum(total * exp2_fast((m - top) * kLog2e));
    if (lane == 0) {                                     // (warps that share a row write the same)
      const float s = a.scores[entry * a.scores_stride + i];
      // the logarithm of the sum's mantissa, 0.7 to 1.4, so that its rounding is one of a small number
      const int up = (int)(__float_as_uint(total * 1.41421356f) >> 23) - 127;
      const float part_of = logf(total * __uint_as_float((uint32_t)(127 - up) << 23));
      norm[i] = s > -CUDART_INF_F ? (double)s - (0.69314718055994531 * up + (double)part_of) : -CUDART_INF;
      peak[i] = top;
    }
  }
  __syncthreads();
  auto score_of = [&](int i, uint32_t key) {             // in 64 bits
    const float v = value_of(key);
    return v == -CUDART_INF_F ? -CUDART_INF : norm[i] + ((double)fminf(v, kFltMax) - (double)peak[i]);
  };
  auto every = [&](auto&& take) {                        // this thread's places, as continuations, list by list while take() says so
    for (int l = list0; l < lists; l += together) {
      const int i = l / p.slices;
      for (int at = place0; at < K; at += g) {
        const unsigned long long place = l == list0 && at == place0 ? early : place_of(l, at);
        if (!place || !take(Next{key_of(score_of(i, (uint32_t)(place >> 32))), place, (uint32_t)i})) break;
      }
    }
  };
  // (bounds are of scores rounded to 32 bits, an order that the rounding keeps)
  float leads = -CUDART_INF_F;
  every([&](const Next& x) {
    leads = fmaxf(leads, (float)value_of(x.score));
    return false;
  });
  float reached = fmaxf(bound_of(leads, K, bounds), bound_of_one(leads, K, bounds_of_one));
  int count;
  for (int i = 0;; ++i) {
    if (leads >= reached && leads > -CUDART_INF_F)
      every([&](const Next& x) {
        const float s = (float)value_of(x.score);
        if (s < reached || s == -CUDART_INF_F) return false;
        const int at = atomicAdd(&listed, 1);
        if (at < kFound) {
          found_score[at] = x.score;
          found_place[at] = x.place;
          found_beam[at] = x.beam;
        }
        return true;
      });
    __syncthreads();
    count = listed;
    if (count <= kFound || i == 2) break;
    // too many (a beam far ahead of the others, whose best lie in few hands): the K-th of those that found room is a better bound
    for (int e = tid; e < kFound; e += kThreads) {
      const unsigned long long mine = found_score[e];
      int at = 0;
#pragma unroll 4
      for (int j = 0; j < kFound; ++j) at += found_score[j] > mine || (found_score[j] == mine && j < e);
      if (at == K - 1) bounds[0] = (float)value_of(mine);
    }
    __syncthreads();
    reached = bounds[0];
    if (tid == 0) listed = 0;
    __syncthreads();
  }
  auto put = [&](int at, const Next& x) {
    const int64_t o = (int64_t)entry * K + at;
    a.out_scores[o] = (float)value_of(x.score);
    a.out_beams[o] = (int)x.beam;
    a.out_tokens[o] = (long long)(uint32_t)~(uint32_t)x.place;
  };
  if (count >= K && count <= kFound) {
    for (int i = tid; i < count; i += kThreads) {
      const Next x{found_score[i], found_place[i], found_beam[i]};
      int at = 0;
#pragma unroll 4
      for (int j = 0; j < count; ++j) at += found_score[j] > x.score;
      for (int j = 0; j < count; ++j)                    // (equal scores, which a short loop is enough to find)
        if (found_score[j] == x.score && j != i) at += before(Next{x.score, found_place[j], found_beam[j]}, x);
      if (at < K) put(at, x);
    }
  } else {
    // too few that are not -infinity, or too many that are equal: the first, the one after it, ...
    Next passed{~0ull, ~0ull, 0}, next{0, 0, 0xffffffffu};
    bool look = true;
    for (int i = 0; i < K; ++i) {
      if (look) {
        next = Next{0, 0, 0xffffffffu};
        every([&](const Next& x) {
          if (!before(passed, x)) return true;
          if (!next.score || before(x, next)) next = x;
          return false;                                  // (the rest of the list comes after it)
        });
      }
      const int from = first_lane(next);
      if (lane == from) heads[warp] = next;
      __syncthreads();
      passed = heads[0];
#pragma unroll
      for (int u = 1; u < kWarps; ++u)
        if (before(heads[u], passed)) passed = heads[u];
      if (tid == 0) put(i, passed);
      look = next.place == passed.place && next.beam == passed.beam;
      __syncthreads();
    }
  }
}

template <class T>
int launch(const pbs_beam_select_t& a, void* workspace, int64_t* bytes, cudaStream_t st) {
  constexpr int N = Piece<T>::N, CHUNK = Row<T>::CHUNK;
  BeamArgs p{};
  p.a = a;
  p.chunks = (int)(((int64_t)a.vocab + N - 1 + CHUNK - 1) / CHUNK);        // (a row may start inside a piece)
  // Segments: so many that all are resident at a time; where there are more rows than that, so short that the CTAs that come last are a small part.
  // (512 rows of 152064 in fp32 in one segment each 64 us, in two 67, in four 73; 64 of 128256 in one 21, in nine 17.)
  const int64_t rows = (int64_t)a.batch * a.beams, resident = (int64_t)kResident * device_sms(), whole = 3 * resident / rows;
  const int64_t slices = rows <= resident ? resident / rows : whole > 1 ? whole : 1;
  p.share = (int)((p.chunks + slices - 1) / slices);
  p.slices = (p.chunks + p.share - 1) / p.share;
  const int64_t ctas = rows * p.slices;
  if (ctas > INT_MAX || (int64_t)p.chunks * CHUNK > INT_MAX) { set_error("beam selection: %lld rows of %d", (long long)rows, a.vocab); return PBS_ERR_SHAPE; }
  if (bytes) {
    *bytes = PBS_PAGED_COUNTER_BYTES + ctas * (8 + 8 * (int64_t)a.keep);
    return PBS_OK;
  }
  p.counters = (unsigned*)workspace;
  p.sums = (float2*)((uint8_t*)workspace + PBS_PAGED_COUNTER_BYTES);
  p.lists = (unsigned long long*)(p.sums + ctas);
  PBS_LAUNCH_EARLY("beam_select_kernel", beam_select_kernel<T>, dim3((unsigned)ctas), kThreads, st, p);
  PBS_CUDA_CHECK_LAUNCH("beam_select_kernel");
  return PBS_OK;
}

int by_type(const pbs_beam_select_t& a, void* workspace, int64_t* bytes, cudaStream_t st) {
  switch (a.dtype) {
    case PBS_BF16: return launch<__nv_bfloat16>(a, workspace, bytes, st);
    case PBS_FP16: return launch<__half>(a, workspace, bytes, st);
    default: return launch<float>(a, workspace, bytes, st);
  }
}

}  // namespace

int beam_select_workspace(const pbs_beam_select_t& a, int64_t* bytes) { return by_type(a, nullptr, bytes, nullptr); }
int launch_beam_select(const pbs_beam_select_t& a, void* workspace, cudaStream_t st) { return by_type(a, workspace, nullptr, st); }

}  // namespace pbs
