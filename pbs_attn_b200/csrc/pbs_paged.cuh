// Paged cache of keys and values: where a token lies, and its codes of 4 bits (layout: include/pbs_b200.h).
#pragma once

#include "pbs_common.cuh"

namespace pbs {

// The C structs as kernels take them.
struct PagedArgs {
  pbs_paged_cache_t c;
  pbs_paged_batch_t b;
  int shift;              // log2(page_size)
  int block_shift;        // 8 bits: log2(block_size)
};

// Strides of a (B, heads, S, D) operand, in elements.
struct RowTensor {
  void* p;
  Strides st;
};

// The word may be host memory: a plain store, any of the faults met will do.
__device__ __forceinline__ void paged_fault(const PagedArgs& a, int what) { *(volatile int32_t*)a.c.status = what; }

// Position of new token i of sequence b; negative where it is left out.
__device__ __forceinline__ int new_position(const pbs_paged_batch_t& b, int seq, int i) {
  const int n = b.new_lens ? min(max(b.new_lens[seq], 0), b.new_tokens) : b.new_tokens;
  return i < n ? b.seq_lens[seq] - n + i : -1;
}

// Page of position pos >= 0 of sequence seq, or -1 (and the fault noted) where there is none.
__device__ __forceinline__ int page_of(const PagedArgs& a, int seq, int pos) {
  const int i = pos >> a.shift;
  if (i >= a.b.max_pages) {
    paged_fault(a, PBS_PAGED_BAD_LENGTH);
    return -1;
  }
  const int page = a.b.block_table[seq * a.b.table_stride + i];
  if ((unsigned)page >= (unsigned)a.c.num_pages) {
    paged_fault(a, PBS_PAGED_BAD_PAGE);
    return -1;
  }
  return page;
}

__device__ __forceinline__ int64_t slot_offset(const int64_t (&st)[3], int page, int head, int slot) {
  return page * st[0] + head * st[1] + slot * st[2];
}

// The kernels of a step are short, and between two of them in a stream 1 to 2 us pass that no kernel runs in.  So each may be put on the SMs while the one
// before it ends: it starts by waiting for that one's results (all threads, before anything else), and lets the next be put there in turn.
// Back to back: selection from four rows 11.2 us a call instead of 13.0, attention of 187 tokens 5.9 instead of 6.8.
__device__ __forceinline__ void after_the_kernel_before() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
inline cudaLaunchAttribute early_launch() {
  cudaLaunchAttribute a = {};
  a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a.val.programmaticStreamSerializationAllowed = 1;
  return a;
}
template <class... P, class... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, int threads, cudaStream_t st, const A&... args) {
  cudaLaunchAttribute early = early_launch();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = st;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}
#define PBS_LAUNCH_EARLY(name, kernel, grid, threads, st, ...)                              \
  do {                                                                                      \
    const cudaError_t launched_ = launch_early(kernel, grid, threads, st, __VA_ARGS__);     \
    if (launched_ != cudaSuccess) return cuda_fail(launched_, name);                        \
  } while (0)

int launch_paged_append(const PagedArgs& a, const RowTensor& k, const RowTensor& v, int q_heads, const RowTensor& q, const RowTensor& qo,
                        const void* cosp, const void* sinp, int64_t cs_b, int64_t cs_s, int table_rows, cudaStream_t st);
int launch_paged_gather(const PagedArgs& a, const RowTensor& k, const RowTensor& v, cudaStream_t st);
int paged_attn_workspace(const PagedArgs& a, int q_heads, int64_t* bytes);
int launch_paged_attn(const PagedArgs& a, int q_heads, const RowTensor& q, const RowTensor& out, float scale, void* workspace, cudaStream_t st);
int launch_paged_reorder(const PagedArgs& a, const pbs_paged_cache_t* const* caches, int layers, int32_t* table, const int32_t* beams, int64_t beams_stride, int n,
                         cudaStream_t st);
int beam_select_workspace(const pbs_beam_select_t& a, int64_t* bytes);
int launch_beam_select(const pbs_beam_select_t& a, void* workspace, cudaStream_t st);
int launch_process_logits(const pbs_logits_t& a, cudaStream_t st);

}  // namespace pbs
