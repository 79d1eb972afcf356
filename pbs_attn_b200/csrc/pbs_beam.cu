// The best continuations of each batch entry's beams: log-softmax of every beam's logits, plus its score, and the K largest of all beams and tokens.
//
// Within a beam the order of the scores is the order of the logits, so one pass over the logits gives both what the softmax needs (their maximum and
// the sum of exponentials) and each slice's K largest; scores are formed for these few only, in 64 bits, when a batch entry's slices meet.
//
// A CTA keeps its slice of a row in registers (up to kMost 16-byte pieces a thread, all loads under way at once).  The K-th largest of a warp's
// 32 largest-of-a-lane is a bound that K of the slice's logits reach; what reaches the best warp's bound (some tens of logits) is listed in shared
// memory and ranked by counting.  Order: (logit, then lower token) as one 64-bit number, so that ties need no case of their own.
// The CTA that finishes an entry last merges the sorted lists of its rows and slices: K times the best of their heads.
#include <climits>
#include <type_traits>

#include "pbs_paged.cuh"

namespace pbs {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMost = 8;                  // 16-byte pieces a thread
constexpr int kResident = 4;              // CTAs a SM
constexpr int kListed = 1024;             // logits that reach the bound; more of them are gone through K times instead
constexpr int kMaxBeams = 32;
constexpr float kFltMax = 3.402823466e38f;
constexpr float kLog2e = 1.44269504f;

struct BeamArgs {
  pbs_beam_select_t a;
  int slices, pieces;                     // of a row; of a thread's share of a slice
  unsigned* counters;                     // by batch entry: slices that are done
  float2* sums;                           // [row][slice]: maximum, sum of exponentials
  unsigned long long* lists;              // [row][slice][keep]
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

// The elements of a 16-byte piece, as floats.
template <class T>
struct Piece;
template <>
struct Piece<float> {
  static constexpr int N = 4;
  static constexpr uint32_t kNever = 0xff800000u;          // -infinity
  static __device__ __forceinline__ void get(const uint4& w, float (&x)[4]) {
    x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ uint32_t bits(const float* p) { return __float_as_uint(*p); }
};
template <>
struct Piece<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr uint32_t kNever = 0xff80ff80u;
  static __device__ __forceinline__ void get(const uint4& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
};
template <>
struct Piece<__half> {
  static constexpr int N = 8;
  static constexpr uint32_t kNever = 0xfc00fc00u;
  static __device__ __forceinline__ void get(const uint4& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
};

__device__ __forceinline__ unsigned long long shfl64(unsigned long long x, int lane) { return __shfl_sync(0xffffffffu, x, lane); }

// Lane k gets the (k + 1)-th largest of the warp's numbers.
__device__ __forceinline__ unsigned long long sorted(unsigned long long x, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const unsigned long long y = __shfl_xor_sync(0xffffffffu, x, j);
      const bool larger = ((lane & j) == 0) == ((lane & k) == 0 || k == 32);
      x = larger ? (x > y ? x : y) : (x < y ? x : y);
    }
  return x;
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

template <class T, int P>
__global__ void __launch_bounds__(kThreads, kResident) beam_select_kernel(const __grid_constant__ BeamArgs p) {
  using E = Piece<T>;
  constexpr int N = E::N;
  const pbs_beam_select_t& a = p.a;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, K = a.keep;
  const int row = blockIdx.x / p.slices, slice = blockIdx.x % p.slices, entry = row / a.beams;
  __shared__ unsigned long long list[kListed];
  __shared__ unsigned long long bounds[kWarps];
  __shared__ float2 part[kWarps];
  __shared__ int listed, last;
  {
    const T* const in = (const T*)a.logits + row * a.logits_stride;
    // pieces are cut where the row's addresses are multiples of 16: `lead` elements before its first
    const int lead = (int)(((uintptr_t)in & 15) / sizeof(T));
    const int first = (slice * P * kThreads + tid) * N - lead;             // vocabulary index of this thread's first piece
    const float own = a.scores[entry * a.scores_stride + row % a.beams];
    const bool alive = own > -CUDART_INF_F;                // (a beam that is not has no order but the tokens')
    uint4 w[P];
#pragma unroll
    for (int k = 0; k < P; ++k) {
      const int v = first + k * kThreads * N;
      w[k] = make_uint4(E::kNever, E::kNever, E::kNever, E::kNever);
      if (!alive) continue;
      if (v >= 0 && v + N <= a.vocab) {
        w[k] = *reinterpret_cast<const uint4*>(in + v);
      } else if (v + N > 0 && v < a.vocab) {
        T* const x = reinterpret_cast<T*>(&w[k]);
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (v + i >= 0 && v + i < a.vocab) x[i] = in[v + i];
      }
    }
    if (tid == 0) listed = 0;
    // this thread's largest, the first of equals, and its sum of exponentials
    float most = -CUDART_INF_F;
    int at = -1;
#pragma unroll
    for (int k = 0; k < P; ++k) {
      float x[N], m;
      E::get(w[k], x);
      m = x[0];
#pragma unroll
      for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
      if (m > most) most = m;
    }
    const float top = fminf(fmaxf(most, -kFltMax), kFltMax);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < P; ++k) {
      float x[N];
      E::get(w[k], x);
#pragma unroll
      for (int i = 0; i < N; ++i) sum += exp2_fast((x[i] - top) * kLog2e);
    }
    if (!(sum <= kFltMax)) {                               // a NaN counts as -infinity, +infinity as the largest number
      sum = 0.f;
#pragma unroll
      for (int k = 0; k < P; ++k) {
        T* const raw = reinterpret_cast<T*>(&w[k]);
        float x[N];
        E::get(w[k], x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (x[i] != x[i]) raw[i] = T(-CUDART_INF_F);
          sum += exp2_fast((fminf(fmaxf(x[i], -kFltMax), kFltMax) - top) * kLog2e);
        }
      }
    }
    unsigned long long best = 0;
#pragma unroll
    for (int k = P - 1; k >= 0; --k) {
      float x[N];
      E::get(w[k], x);
#pragma unroll
      for (int i = N - 1; i >= 0; --i) {
        const int v = first + k * kThreads * N + i;
        if (x[i] == most && v >= 0 && v < a.vocab) at = v;
      }
    }
    if (at >= 0) best = ordered(most, at);
    // the slice's maximum and sum
    const float wide = warp_max(top);
    sum = warp_sum(sum * exp2_fast((top - wide) * kLog2e));
    if (lane == 0) part[warp] = make_float2(wide, sum);
    // bound: K of a warp's lanes, or of two warps', hold a logit that reaches it
    const unsigned long long order = sorted(best, lane), kth = shfl64(order, min(K, 32) - 1);
    if (lane == 0) bounds[warp] = kth;
    __syncthreads();
    unsigned long long bound = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const unsigned long long b = K <= 32 ? bounds[i] : bounds[i] < bounds[i ^ 1] ? bounds[i] : bounds[i ^ 1];
      bound = b > bound ? b : bound;
    }
    const float least = bound ? value_of((uint32_t)(bound >> 32)) : -CUDART_INF_F;
    if (best >= bound && best != 0) {
#pragma unroll
      for (int k = 0; k < P; ++k) {
        float x[N];
        E::get(w[k], x);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int v = first + k * kThreads * N + i;
          if (!(x[i] >= least) || v < 0 || v >= a.vocab) continue;
          const unsigned long long o = ordered(x[i], v);
          if (o < bound) continue;
          const int n = atomicAdd(&listed, 1);
          if (n < kListed) list[n] = o;
        }
      }
    }
    __syncthreads();
    unsigned long long* const out = p.lists + (int64_t)blockIdx.x * K;
    if (tid == 0) {
      float2 all = part[0];
#pragma unroll
      for (int i = 1; i < kWarps; ++i) {
        const float m = fmaxf(all.x, part[i].x);
        all = make_float2(m, all.y * exp2_fast((all.x - m) * kLog2e) + part[i].y * exp2_fast((part[i].x - m) * kLog2e));
      }
      p.sums[blockIdx.x] = all;
    }
    const int n = listed;
    if (n <= kListed) {
      for (int i = tid; i < n; i += kThreads) {
        const unsigned long long mine = list[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += list[j] > mine;
        if (rank < K) out[rank] = mine;
      }
      for (int i = n + tid; i < K; i += kThreads) out[i] = 0;              // (a slice of fewer tokens)
    } else {                                               // very many in few lanes: the largest, the one after it, ...
      unsigned long long lower = ~0ull;
      for (int r = 0; r < K; ++r) {
        unsigned long long mine = 0;
#pragma unroll
        for (int k = 0; k < P; ++k) {
          float x[N];
          E::get(w[k], x);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int v = first + k * kThreads * N + i;
            if (v < 0 || v >= a.vocab) continue;
            const unsigned long long o = ordered(x[i], v);
            if (o < lower && o > mine) mine = o;
          }
        }
        mine = shfl64(sorted(mine, lane), 0);
        if (lane == 0) list[warp] = mine;
        __syncthreads();
        mine = list[0];
#pragma unroll
        for (int i = 1; i < kWarps; ++i) mine = list[i] > mine ? list[i] : mine;
        if (tid == 0) out[r] = mine;
        lower = mine;
        __syncthreads();
      }
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
  }
  __syncthreads();
  if (!last) return;

  // the entry's rows and slices meet: lists of one entry are neighbours
  __shared__ double norm[kMaxBeams];                       // of a beam: its score, less the logarithm of its sum
  __shared__ float peak[kMaxBeams];
  __shared__ Next heads[kWarps];
  const int rows = a.beams, lists = rows * p.slices;
  const int64_t base = (int64_t)entry * lists;
  for (int r = warp; r < rows; r += kWarps) {
    float m = -kFltMax;
    for (int s = lane; s < p.slices; s += 32) m = fmaxf(m, __ldcg(&p.sums[base + r * p.slices + s]).x);
    m = warp_max(m);
    double sum = 0.0;
    for (int s = lane; s < p.slices; s += 32) {
      const float2 x = __ldcg(&p.sums[base + r * p.slices + s]);
      sum += (double)x.y * (double)exp2_fast((x.x - m) * kLog2e);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      const float own = a.scores[entry * a.scores_stride + r];
      norm[r] = own > -CUDART_INF_F ? (double)own - log(sum) : -CUDART_INF;
      peak[r] = m;
    }
  }
  __syncthreads();
  auto next = [&](int l, int i) {                          // entry i of list l
    Next x{0, 0, 0xffffffffu};
    if (i < K) x.place = __ldcg(p.lists + (base + l) * K + i);
    if (x.place) {
      x.beam = l / p.slices;
      const float v = value_of((uint32_t)(x.place >> 32));
      // (the largest number stands for infinity)
      const double score = v == -CUDART_INF_F ? -CUDART_INF : norm[x.beam] + ((double)fminf(v, kFltMax) - (double)peak[x.beam]);
      x.score = key_of(score);
    }
    return x;
  };
  // a thread's lists l = tid, tid + kThreads, ...: how far each has been taken, in shared memory
  uint8_t* const taken = reinterpret_cast<uint8_t*>(list);
  const bool many = lists > kListed * 8;                   // (more lists than there is room for are looked through anew each time)
  if (!many)
    for (int l = tid; l < lists; l += kThreads) taken[l] = 0;
  Next mine{0, 0, 0xffffffffu}, floor_{~0ull, ~0ull, 0};
  int mine_list = -1;
  auto look = [&] {                                        // the best of this thread's lists
    mine = Next{0, 0, 0xffffffffu};
    for (int l = tid; l < lists; l += kThreads) {
      Next x{0, 0, 0xffffffffu};
      if (!many) {
        x = next(l, taken[l]);
      } else {
        for (int i = 0; i < K; ++i) {
          x = next(l, i);
          if (!x.place || before(floor_, x)) break;
        }
      }
      if (x.place && (!mine.place || before(x, mine))) {
        mine = x;
        mine_list = l;
      }
    }
  };
  auto head = [&] {                                        // the best of the warp's
    const int l = first_lane(mine);
    if (lane == l) heads[warp] = mine;
  };
  look();
  head();
  __syncthreads();
  for (int r = 0; r < K; ++r) {
    int w = 0;
    Next x = heads[0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i)
      if (before(heads[i], x)) {
        x = heads[i];
        w = i;
      }
    __syncthreads();
    if (tid == 0) {
      const int64_t o = (int64_t)entry * K + r;
      a.out_scores[o] = (float)value_of(x.score);
      a.out_beams[o] = (int)x.beam;
      a.out_tokens[o] = (long long)(uint32_t)~(uint32_t)x.place;
    }
    floor_ = x;
    if (warp == w) {
      if (mine.place == x.place && mine.beam == x.beam && mine_list >= 0) {
        if (!many) ++taken[mine_list];
        look();
      }
      __syncwarp();
      head();
    }
    __syncthreads();
  }
}

template <class T>
constexpr int elements() { return 16 / (int)sizeof(T); }

// Pieces of a thread (a power of two) and slices of a row: as many slices as are resident at a time, though no smaller than a piece a
// thread, and as many more as it takes to keep them in registers.
template <class T>
void cut(const pbs_beam_select_t& a, int* slices, int* pieces) {
  const int64_t per = (int64_t)kThreads * elements<T>(), total = ((int64_t)a.vocab + elements<T>() - 1 + per - 1) / per;
  const int64_t rows = (int64_t)a.batch * a.beams, fit = (int64_t)kResident * device_sms() / rows;
  int64_t p = (total + (fit > 1 ? fit : 1) - 1) / (fit > 1 ? fit : 1);
  *pieces = p <= 1 ? 1 : p <= 2 ? 2 : p <= 4 ? 4 : kMost;
  *slices = (int)((total + *pieces - 1) / *pieces);
}

template <class T>
int launch(const pbs_beam_select_t& a, void* workspace, int64_t* bytes, cudaStream_t st) {
  BeamArgs p{};
  p.a = a;
  cut<T>(a, &p.slices, &p.pieces);
  const int64_t ctas = (int64_t)a.batch * a.beams * p.slices;
  if (ctas > INT_MAX) { set_error("beam selection: %lld rows of %d", (long long)a.batch * a.beams, a.vocab); return PBS_ERR_SHAPE; }
  if (bytes) {
    *bytes = PBS_PAGED_COUNTER_BYTES + ctas * (8 + 8 * (int64_t)a.keep);
    return PBS_OK;
  }
  p.counters = (unsigned*)workspace;
  p.sums = (float2*)((uint8_t*)workspace + PBS_PAGED_COUNTER_BYTES);
  p.lists = (unsigned long long*)(p.sums + ctas);
  const dim3 grid((unsigned)ctas);
  switch (p.pieces) {
    case 1: beam_select_kernel<T, 1><<<grid, kThreads, 0, st>>>(p); break;
    case 2: beam_select_kernel<T, 2><<<grid, kThreads, 0, st>>>(p); break;
    case 4: beam_select_kernel<T, 4><<<grid, kThreads, 0, st>>>(p); break;
    default: beam_select_kernel<T, kMost><<<grid, kThreads, 0, st>>>(p); break;
  }
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
