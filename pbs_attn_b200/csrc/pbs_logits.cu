// Penalties for repeated tokens, biases and a grammar mask on the logits of a step, in one pass.
//
// A CTA owns a slice of one row's vocabulary.  It counts the row's history into shared memory (one word per token: how often written, whether
// in the prompt, whether a bias names it), then streams the slice once.  Counting anew in each step keeps no state between calls, so rows can
// be reordered, dropped and rolled back freely.
#include "pbs_paged.cuh"

namespace pbs {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kInPrompt = 1u << 31, kBiased = 1u << 30, kCount = kBiased - 1;

__device__ __forceinline__ int64_t id_at(const void* p, int bytes, int64_t i) {
  return bytes == 8 ? ((const long long*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

template <int DT>
__global__ void __launch_bounds__(kThreads) logits_kernel(const __grid_constant__ pbs_logits_t a, int slice_chunks) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int EPV = 16 / (int)sizeof(T);
  extern __shared__ uint32_t seen[];
  const int row = blockIdx.y;
  const T* in = (const T*)a.logits + row * a.logits_stride;
  T* out = (T*)a.out + row * a.out_stride;
  // 16-byte pieces are cut where the row's addresses are multiples of 16: `lead` elements before its first
  const int lead = (int)(((uintptr_t)in & 15) / sizeof(T));
  const bool wide = ((uintptr_t)in & 15) == ((uintptr_t)out & 15);
  const int first = blockIdx.x * slice_chunks * EPV - lead;              // vocabulary index of seen[0]
  const int lo = max(first, 0), hi = min(first + slice_chunks * EPV, a.vocab);
  if (lo >= hi) return;
  const float rep = a.repetition ? a.repetition[row] : a.repetition_all, freq = a.frequency ? a.frequency[row] : a.frequency_all;
  const float pres = a.presence ? a.presence[row] : a.presence_all;
  const bool counts = a.tokens && (rep != 1.f || freq != 0.f || pres != 0.f), biased = a.bias_ids != nullptr;
  if (counts || biased) {
    for (int i = threadIdx.x; i < hi - first; i += kThreads) seen[i] = 0;
    __syncthreads();
    if (counts) {
      const int n = a.token_lens ? min(max(a.token_lens[row], 0), a.history) : a.history;
      const int prompt = a.prompt_lens ? a.prompt_lens[row] : 0;
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const int64_t id = id_at(a.tokens, a.token_bytes, row * a.tokens_stride + i);
        if (id < lo || id >= hi) continue;
        if (i < prompt) atomicOr(&seen[id - first], kInPrompt);
        else atomicAdd(&seen[id - first], 1u);
      }
    }
    if (biased) {
      __syncthreads();
      for (int i = threadIdx.x; i < a.biases; i += kThreads) {
        const int64_t id = id_at(a.bias_ids, a.bias_id_bytes, row * a.bias_ids_stride + i);
        if (id >= lo && id < hi) atomicOr(&seen[id - first], kBiased);
      }
    }
    __syncthreads();
  }
  const uint32_t* allowed = a.allowed ? a.allowed + row * a.allowed_stride : nullptr;
  auto process = [&](float x, int v) {
    if (counts || biased) {
      const uint32_t w = seen[v - first];
      if (w) {
        const float c = (float)(w & kCount);
        if (w & (kInPrompt | kCount)) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        if (w & kCount) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, c)), pres);
        if (w & kBiased) {
          float sum = 0.f;
          for (int i = 0; i < a.biases; ++i)
            if (id_at(a.bias_ids, a.bias_id_bytes, row * a.bias_ids_stride + i) == v) sum += a.bias_values[row * a.bias_values_stride + i];
          x = __fadd_rn(x, sum);
        }
      }
    }
    if (allowed && !((allowed[v >> 5] >> (v & 31)) & 1)) x = -CUDART_INF_F;
    return E::cvt(x);
  };
  for (int s = threadIdx.x; s * EPV < hi - first; s += kThreads) {
    const int v0 = first + s * EPV;
    if (wide && v0 >= lo && v0 + EPV <= hi) {
      uint4 w = *reinterpret_cast<const uint4*>(in + v0);
      T* x = reinterpret_cast<T*>(&w);
#pragma unroll
      for (int e = 0; e < EPV; ++e) x[e] = process(E::ld(x + e), v0 + e);
      *reinterpret_cast<uint4*>(out + v0) = w;
    } else {
      for (int v = max(v0, lo); v < min(v0 + EPV, hi); ++v) out[v] = process(E::ld(in + v), v);
    }
  }
}

template <int DT>
int launch(const pbs_logits_t& a, cudaStream_t st) {
  constexpr int EPV = 16 / (int)sizeof(typename Elem<DT>::T);
  constexpr int kSlice = 4096;
  const dim3 grid((unsigned)((a.vocab + EPV - 1 + kSlice - 1) / kSlice), (unsigned)a.rows);   // (EPV - 1: the row may start inside a piece)
  logits_kernel<DT><<<grid, kThreads, kSlice * 4, st>>>(a, kSlice / EPV);
  PBS_CUDA_CHECK_LAUNCH("logits_kernel");
  return PBS_OK;
}

}  // namespace

int launch_process_logits(const pbs_logits_t& a, cudaStream_t st) {
  switch (a.dtype) {
    case PBS_BF16: return launch<PBS_BF16>(a, st);
    case PBS_FP16: return launch<PBS_FP16>(a, st);
    default: return launch<PBS_FP32>(a, st);
  }
}

}  // namespace pbs
