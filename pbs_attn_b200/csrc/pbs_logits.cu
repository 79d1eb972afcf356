// Penalties for repeated tokens, biases and a grammar mask on the logits of a step, in one pass.
//
// A CTA owns a slice of one row's vocabulary.  Half of its warps stream the slice and mask it; the other half meanwhile count the row's
// history into shared memory (an entry per token: how often written, whether in the prompt, whether a bias names it) and list the tokens
// met; then all go over the listed tokens, which are few, and penalise what is not masked.  One after the other in the same warps the
// three took 44 us for 64 rows of 152064 in fp32, side by side 21 (the stream alone 17).
// Counting anew in each step keeps no state between calls, so rows can be reordered, dropped and rolled back freely.
//
// Large batches are bound by how the slices fall on the SMs and by half of the warps streaming: 64 rows of 152064 in fp32 with histories of up to
// 8192 take 20.8 us, 3.9 TB/s, 60 % of the copy rate (four slices a row, 256 CTAs, on 296 places); single rows by latency: 128256 in bf16 4.9 us.
// More than kBiases biases in a slice, and logits and result at different distances from 16 bytes, work and are slow: the former reads all of the
// row's biases for each listed token, the latter goes element by element.
#include <climits>

#include "pbs_paged.cuh"

namespace pbs {
namespace {

constexpr int kHalf = 256, kThreads = 2 * kHalf;
constexpr int kAhead = 8;                 // 16-byte pieces that a thread has under way
constexpr int kIds = 8;                   // ids that it has
constexpr int kListed = 2048, kBiases = 256;
constexpr int kResident = 2;              // CTAs a SM

// Entries of 16 bits wherever a count cannot outgrow 14 of them, i.e. for histories below 2^14; else of 32.
template <class W>
struct Entry {
  static constexpr int BITS = 8 * (int)sizeof(W);
  static constexpr uint32_t kInPrompt = 1u << (BITS - 1), kBiased = 1u << (BITS - 2), kCount = kBiased - 1;
  static constexpr int kMostSlice = 96 * 1024 / (int)sizeof(W);
  // Marks or counts entry i; true for the first to touch it.
  static __device__ __forceinline__ bool mark(W* e, int i, uint32_t bit) {
    if constexpr (BITS == 32) return atomicOr(reinterpret_cast<uint32_t*>(e) + i, bit) == 0;
    else return (atomicOr(reinterpret_cast<uint32_t*>(e) + i / 2, bit << i % 2 * 16) >> i % 2 * 16 & 0xffff) == 0;
  }
  static __device__ __forceinline__ bool count(W* e, int i) {
    if constexpr (BITS == 32) return atomicAdd(reinterpret_cast<uint32_t*>(e) + i, 1u) == 0;
    else return (atomicAdd(reinterpret_cast<uint32_t*>(e) + i / 2, 1u << i % 2 * 16) >> i % 2 * 16 & 0xffff) == 0;
  }
};

__device__ __forceinline__ int64_t id_at(const void* p, int bytes, int64_t i) {
  return bytes == 8 ? ((const long long*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

template <int DT, class W>
__global__ void __launch_bounds__(kThreads, kResident) logits_kernel(const __grid_constant__ pbs_logits_t a, int slice) {
  using E = Elem<DT>;
  using T = typename E::T;
  using N = Entry<W>;
  constexpr int EPV = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) uint8_t smem[];
  W* const seen = reinterpret_cast<W*>(smem);
  __shared__ int listed[kListed];                          // tokens met, as entries
  __shared__ int2 biases[kBiases];                         // biases of this slice: index in the row, entry
  __shared__ int n_listed, n_biases;
  const int row = blockIdx.y, tid = threadIdx.x % kHalf;
  const bool streams = threadIdx.x < kHalf;
  const T* in = (const T*)a.logits + row * a.logits_stride;
  T* out = (T*)a.out + row * a.out_stride;
  // 16-byte pieces are cut where the row's addresses are multiples of 16: `lead` elements before its first
  const int lead = (int)(((uintptr_t)in & 15) / sizeof(T));
  const int first = blockIdx.x * slice - lead;             // vocabulary index of seen[0]
  const int lo = max(first, 0), hi = min(first + slice, a.vocab);
  if (lo >= hi) return;
  const uint32_t* allowed = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
  const float rep = a.repetition ? a.repetition[row] : a.repetition_all, freq = a.frequency ? a.frequency[row] : a.frequency_all;
  const float pres = a.presence ? a.presence[row] : a.presence_all;
  const bool counts = a.tokens && (rep != 1.f || freq != 0.f || pres != 0.f), biased = a.bias_ids != nullptr;
  const int64_t bias_row = row * a.bias_ids_stride;

  if (streams) {
    const T never = E::cvt(-CUDART_INF_F);
    const bool wide = ((uintptr_t)in & 15) == ((uintptr_t)out & 15);
    for (int s0 = tid * EPV; s0 < hi - first; s0 += kAhead * kHalf * EPV) {
      uint4 now[kAhead];
      uint32_t may[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int v0 = first + s0 + k * kHalf * EPV;
        const bool whole = wide && v0 >= lo && v0 + EPV <= hi;
        if (whole) now[k] = *reinterpret_cast<const uint4*>(in + v0);
        may[k] = whole && allowed ? allowed[v0 >> 5] : 0;             // (the words as they are: using one here would wait for it)
      }
      if (lead != 0 && allowed) {                                     // a piece's bits may lie in two words
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int v0 = first + s0 + k * kHalf * EPV;
          if (wide && v0 >= lo && v0 + EPV <= hi)
            may[k] = __funnelshift_r(may[k], (v0 & 31) + EPV > 32 ? allowed[(v0 >> 5) + 1] : 0u, v0 & 31);
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int v0 = first + s0 + k * kHalf * EPV;
        if (wide && v0 >= lo && v0 + EPV <= hi) {
          T* x = reinterpret_cast<T*>(&now[k]);
          if (allowed) {
            const uint32_t bits = lead != 0 ? may[k] : may[k] >> (v0 & 31);
#pragma unroll
            for (int i = 0; i < EPV; ++i)
              if (!(bits >> i & 1)) x[i] = never;
          }
          *reinterpret_cast<uint4*>(out + v0) = now[k];
        } else {
          for (int v = max(v0, lo); v < min(v0 + EPV, hi); ++v) out[v] = allowed && !(allowed[v >> 5] >> (v & 31) & 1) ? never : in[v];
        }
      }
    }
  } else if (counts || biased) {
    const int n = !counts ? 0 : a.token_lens ? min(max(a.token_lens[row], 0), a.history) : a.history;
    const int prompt = a.prompt_lens ? min(max(a.prompt_lens[row], 0), n) : 0;           // (any number is taken: "all of it" may be 2^31 - 1)
    const int words = ((hi - first) * (int)sizeof(W) + 15) / 16;
    for (int i = tid; i < words; i += kHalf) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) n_listed = n_biases = 0;
    asm volatile("bar.sync 1, %0;" ::"n"(kHalf) : "memory");             // (of these warps)
    auto list = [&](bool fresh, int entry) {
      if (!fresh) return;
      const int at = atomicAdd(&n_listed, 1);
      if (at < kListed) listed[at] = entry;
    };
    const bool wide_ids = a.token_bytes == 8;
    const int64_t base = row * a.tokens_stride;
    for (int i = tid + (rep == 1.f ? prompt : 0); i < n; i += kIds * kHalf) {       // (the prompt is for the repetition penalty only)
      int64_t id[kIds];
      if (wide_ids) {
#pragma unroll
        for (int k = 0; k < kIds; ++k) id[k] = i + k * kHalf < n ? ((const long long*)a.tokens)[base + i + k * kHalf] : -1;
      } else {
#pragma unroll
        for (int k = 0; k < kIds; ++k) id[k] = i + k * kHalf < n ? ((const int32_t*)a.tokens)[base + i + k * kHalf] : -1;
      }
#pragma unroll
      for (int k = 0; k < kIds; ++k) {
        if (id[k] < lo || id[k] >= hi) continue;
        const int entry = (int)id[k] - first;
        list(i + k * kHalf < prompt ? N::mark(seen, entry, N::kInPrompt) : N::count(seen, entry), entry);
      }
    }
    for (int i = tid; biased && i < a.biases; i += kHalf) {
      const int64_t id = id_at(a.bias_ids, a.bias_id_bytes, bias_row + i);
      if (id < lo || id >= hi) continue;
      const int entry = (int)id - first, at = atomicAdd(&n_biases, 1);
      if (at < kBiases) biases[at] = make_int2(i, entry);
      list(N::mark(seen, entry, N::kBiased), entry);
    }
  }
  if (!counts && !biased) return;
  __syncthreads();                                         // the slice is in `out`, masked

  auto penalise = [&](int entry) {
    const int v = first + entry;
    const uint32_t w = seen[entry];
    if (!w || (allowed && !(allowed[v >> 5] >> (v & 31) & 1))) return;
    float x = E::ld(out + v);
    const float c = (float)(w & N::kCount);
    if (w & (N::kInPrompt | N::kCount)) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    if (w & N::kCount) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, c)), pres);
    if (w & N::kBiased) {                                  // the values listed for it, added in their order
      float sum = 0.f;
      if (n_biases > kBiases) {
        for (int i = 0; i < a.biases; ++i)
          if (id_at(a.bias_ids, a.bias_id_bytes, bias_row + i) == v) sum += a.bias_values[row * a.bias_values_stride + i];
      } else {
        for (int last = -1;;) {                            // (the list is in any order)
          int at = INT_MAX;
          for (int i = 0; i < n_biases; ++i)
            if (biases[i].y == entry && biases[i].x > last) at = min(at, biases[i].x);
          if (at == INT_MAX) break;
          sum += a.bias_values[row * a.bias_values_stride + at];
          last = at;
        }
      }
      x = __fadd_rn(x, sum);
    }
    out[v] = E::cvt(x);
  };
  if (n_listed <= kListed)
    for (int i = threadIdx.x; i < n_listed; i += kThreads) penalise(listed[i]);
  else
    for (int i = threadIdx.x; i < hi - first; i += kThreads) penalise(i);
}

template <int DT, class W>
int launch(const pbs_logits_t& a, cudaStream_t st) {
  constexpr int EPV = 16 / (int)sizeof(typename Elem<DT>::T);
  // As many slices as are resident at a time (every slice reads the row's history), though no smaller than a piece a thread and no
  // larger than the entries that leave room for kResident CTAs.
  const int64_t span = (int64_t)a.vocab + EPV - 1;         // (the row may start inside a piece)
  const int64_t fit = kResident * device_sms() / a.rows, least = kHalf * EPV;
  int64_t slice = (span + (fit > 1 ? fit : 1) - 1) / (fit > 1 ? fit : 1);
  slice = (slice < least ? least : slice > Entry<W>::kMostSlice ? Entry<W>::kMostSlice : slice) + 15 & ~15ll;
  const dim3 grid((unsigned)((span + slice - 1) / slice), (unsigned)a.rows);
  const int bytes = (int)slice * (int)sizeof(W);
  if (bytes > 32 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(logits_kernel<DT, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024);
    if (e != cudaSuccess) return cuda_fail(e, "logits_kernel shared memory");
  }
  logits_kernel<DT, W><<<grid, kThreads, bytes, st>>>(a, (int)slice);
  PBS_CUDA_CHECK_LAUNCH("logits_kernel");
  return PBS_OK;
}

template <int DT>
int by_history(const pbs_logits_t& a, cudaStream_t st) {
  return a.history < 1 << 14 ? launch<DT, uint16_t>(a, st) : launch<DT, uint32_t>(a, st);
}

}  // namespace

int launch_process_logits(const pbs_logits_t& a, cudaStream_t st) {
  switch (a.dtype) {
    case PBS_BF16: return by_history<PBS_BF16>(a, st);
    case PBS_FP16: return by_history<PBS_FP16>(a, st);
    default: return by_history<PBS_FP32>(a, st);
  }
}

}  // namespace pbs
