// Paged cache of keys and values: where a token lies, and its codes of 4 bits (layout: include/pbs_b200.h).
#pragma once

#include "pbs_common.cuh"

namespace pbs {

// The C structs as kernels take them.
struct PagedArgs {
  pbs_paged_cache_t c;
  pbs_paged_batch_t b;
  int shift;              // log2(page_size)
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

int launch_paged_append(const PagedArgs& a, const RowTensor& k, const RowTensor& v, int q_heads, const RowTensor& q, const RowTensor& qo,
                        const void* cosp, const void* sinp, int64_t cs_b, int64_t cs_s, int table_rows, cudaStream_t st);
int launch_paged_gather(const PagedArgs& a, const RowTensor& k, const RowTensor& v, cudaStream_t st);
int paged_attn_workspace(const PagedArgs& a, int q_heads, int64_t* bytes);
int launch_paged_attn(const PagedArgs& a, int q_heads, const RowTensor& q, const RowTensor& out, float scale, void* workspace, cudaStream_t st);
int launch_process_logits(const pbs_logits_t& a, cudaStream_t st);

}  // namespace pbs
