// extern "C" entry points of what follows a prompt: paged cache, attention over it, logits of a step.
#include <climits>

#include "pbs_paged.cuh"

namespace pbs {
namespace {

int check_pages(const char* name, const void* p, const int64_t (&st)[3], int bytes, int align) {
  PBS_NONNULL(p);
  bool ok = ((uintptr_t)p % align) == 0;
  for (int i = 0; i < 3; ++i) ok = ok && st[i] >= 0 && (st[i] * bytes) % align == 0;
  if (!ok) { set_error("%s: the pool and every token's row must start on a multiple of %d bytes, strides must not be negative", name, align); return PBS_ERR_LAYOUT; }
  return PBS_OK;
}

int check_paged(const pbs_paged_cache_t* c, const pbs_paged_batch_t* b, PagedArgs* out) {
  PBS_NONNULL(c);
  PBS_NONNULL(b);
  if (c->dtype != PBS_BF16 && c->dtype != PBS_FP16) { set_error("paged cache: dtype %d is not bf16/fp16", c->dtype); return PBS_ERR_ARG; }
  if (c->bits != 16 && c->bits != 8 && c->bits != 4) { set_error("paged cache: %d bits, need 16, 8 or 4", c->bits); return PBS_ERR_ARG; }
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) { set_error("paged cache: head_dim %d, need 64, 128 or 256", c->head_dim); return PBS_ERR_SHAPE; }
  if (c->bits == 4 && c->group_size != 32 && c->group_size != 64) { set_error("paged cache: group_size %d, need 32 or 64", c->group_size); return PBS_ERR_SHAPE; }
  if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1))) { set_error("paged cache: page_size %d, need a power of two in [16, 1024]", c->page_size); return PBS_ERR_SHAPE; }
  if (c->bits == 8 && ((c->block_size != 16 && c->block_size != 32 && c->block_size != 64) || c->block_size > c->page_size)) {
    set_error("paged cache: block_size %d, need 16, 32 or 64 and at most page_size (%d)", c->block_size, c->page_size);
    return PBS_ERR_ARG;
  }
  if (c->num_pages < 1 || c->kv_heads < 1) { set_error("paged cache: %d pages, %d heads", c->num_pages, c->kv_heads); return PBS_ERR_SHAPE; }
  if (b->batch < 1 || b->new_tokens < 1 || b->max_pages < 1) {
    set_error("batch, new_tokens and max_pages must be positive (got %d, %d, %d)", b->batch, b->new_tokens, b->max_pages);
    return PBS_ERR_SHAPE;
  }
  if ((int64_t)b->max_pages * c->page_size > INT_MAX - (1 << 20)) { set_error("a row of the block table holds 2^31 tokens or more"); return PBS_ERR_SHAPE; }
  if (b->table_stride < 0) { set_error("block_table: negative stride"); return PBS_ERR_LAYOUT; }
  if (b->batch > 4096) { set_error("%d sequences in a call, at most 4096", b->batch); return PBS_ERR_SHAPE; }
  PBS_NONNULL(b->block_table);
  PBS_NONNULL(b->seq_lens);
  PBS_NONNULL(c->status);
  PBS_TRY(check_pages("k pages", c->k, c->k_strides, c->bits == 16 ? 2 : 1, 16));
  PBS_TRY(check_pages("v pages", c->v, c->v_strides, c->bits == 16 ? 2 : 1, 16));
  if (c->bits == 4) {
    const int row = 4 * (c->head_dim / c->group_size), align = row < 16 ? row : 16;
    PBS_TRY(check_pages("k_params", c->k_params, c->k_params_strides, 2, align));
    PBS_TRY(check_pages("v_params", c->v_params, c->v_params_strides, 2, align));
  }
  if (c->bits == 8) {
    PBS_TRY(check_pages("k_params", c->k_params, c->k_params_strides, 4, 4));
    PBS_TRY(check_pages("v_params", c->v_params, c->v_params_strides, 4, 4));
  }
  out->c = *c;
  out->b = *b;
  out->shift = 0;
  while ((1 << out->shift) < c->page_size) ++out->shift;
  out->block_shift = c->bits != 8 ? 0 : c->block_size == 16 ? 4 : c->block_size == 32 ? 5 : 6;
  return PBS_OK;
}

int check_rows(const char* name, const PagedArgs& a, int heads, const void* p, const int64_t* st, bool written, RowTensor* out) {
  PBS_TRY(check_tensor(name, p, st, a.c.dtype, &out->st));
  if (written && ((heads > 1 && st[1] == 0) || (a.b.batch > 1 && st[0] == 0))) { set_error("%s: written rows share memory (zero stride)", name); return PBS_ERR_LAYOUT; }
  out->p = const_cast<void*>(p);
  return PBS_OK;
}

int check_count(const PagedArgs& a, int64_t heads) {
  if ((int64_t)a.b.batch * a.b.new_tokens * heads > INT_MAX || heads > 65535) { set_error("more than 2^31 rows in a call, or 65535 heads"); return PBS_ERR_SHAPE; }
  return PBS_OK;
}

int check_beams(const pbs_beam_select_t* a) {
  PBS_NONNULL(a);
  if (a->dtype < PBS_BF16 || a->dtype > PBS_FP32) { set_error("dtype %d is not bf16/fp16/fp32", a->dtype); return PBS_ERR_ARG; }
  if (a->batch < 1 || a->batch > 1024 || a->beams < 1 || a->beams > 32 || a->vocab < 1 || a->vocab > (1 << 30)) {
    set_error("beam selection: %d entries (1 .. 1024) of %d beams (1 .. 32) of %d tokens", a->batch, a->beams, a->vocab);
    return PBS_ERR_SHAPE;
  }
  if (a->keep < 1 || a->keep > 64 || a->keep > (int64_t)a->beams * a->vocab) { set_error("beam selection: keep %d, need 1 .. 64 and no more than there are", a->keep); return PBS_ERR_SHAPE; }
  PBS_NONNULL(a->logits);
  PBS_NONNULL(a->scores);
  PBS_NONNULL(a->out_scores);
  PBS_NONNULL(a->out_beams);
  PBS_NONNULL(a->out_tokens);
  if ((uintptr_t)a->logits % elem_bytes(a->dtype) || a->logits_stride < 0 || a->scores_stride < 0 || ((uintptr_t)a->scores | (uintptr_t)a->out_scores | (uintptr_t)a->out_beams) % 4 ||
      (uintptr_t)a->out_tokens % 8) {
    set_error("beam selection: pointers must be aligned to their elements, strides must not be negative");
    return PBS_ERR_LAYOUT;
  }
  return PBS_OK;
}

int check_q_heads(const PagedArgs& a, int q_heads) {
  if (q_heads < 1 || q_heads % a.c.kv_heads) { set_error("kv_heads %d does not divide q_heads %d", a.c.kv_heads, q_heads); return PBS_ERR_SHAPE; }
  return check_count(a, q_heads);
}

}  // namespace
}  // namespace pbs

using namespace pbs;

extern "C" {

int pbs_paged_append(const pbs_paged_cache_t* cache, const pbs_paged_batch_t* batch, const void* k, const int64_t k_strides[4],
                     const void* v, const int64_t v_strides[4], int32_t q_heads, const void* q, const int64_t q_strides[4], void* q_out,
                     const int64_t q_out_strides[4], const void* cos_table, const void* sin_table, const int64_t cs_strides[3],
                     int32_t table_rows, void* stream) {
  PagedArgs a;
  RowTensor kt, vt, qt{}, ot{};
  PBS_TRY(check_paged(cache, batch, &a));
  PBS_TRY(check_rows("k", a, a.c.kv_heads, k, k_strides, false, &kt));
  PBS_TRY(check_rows("v", a, a.c.kv_heads, v, v_strides, false, &vt));
  if ((cos_table == nullptr) != (sin_table == nullptr)) { set_error("cos and sin come together"); return PBS_ERR_ARG; }
  int64_t cs_b = 0, cs_s = 0;
  if (cos_table) {
    PBS_NONNULL(cs_strides);
    if (cs_strides[2] != 1 || cs_strides[0] < 0 || cs_strides[1] < 0 || ((cs_strides[0] | cs_strides[1]) * 2) % 16 ||
        ((uintptr_t)cos_table | (uintptr_t)sin_table) % 16) {
      set_error("cos / sin: rows must be dense and start on 16-byte boundaries");
      return PBS_ERR_LAYOUT;
    }
    if (table_rows < 0) { set_error("table_rows %d", table_rows); return PBS_ERR_SHAPE; }
    cs_b = cs_strides[0];
    cs_s = cs_strides[1];
  }
  if (q) {
    if (!cos_table) { set_error("queries are given but no rotary tables"); return PBS_ERR_ARG; }
    PBS_TRY(check_q_heads(a, q_heads));
    PBS_TRY(check_rows("q", a, q_heads, q, q_strides, false, &qt));
    PBS_TRY(check_rows("q_out", a, q_heads, q_out, q_out_strides, true, &ot));
  } else {
    q_heads = 0;
  }
  PBS_TRY(check_count(a, q_heads + 2ll * a.c.kv_heads));
  return launch_paged_append(a, kt, vt, q_heads, qt, ot, cos_table, sin_table, cs_b, cs_s, table_rows, (cudaStream_t)stream);
}

int pbs_paged_gather(const pbs_paged_cache_t* cache, const pbs_paged_batch_t* batch, void* k, const int64_t k_strides[4], void* v,
                     const int64_t v_strides[4], void* stream) {
  PagedArgs a;
  RowTensor kt, vt;
  PBS_TRY(check_paged(cache, batch, &a));
  PBS_TRY(check_rows("k", a, a.c.kv_heads, k, k_strides, true, &kt));
  PBS_TRY(check_rows("v", a, a.c.kv_heads, v, v_strides, true, &vt));
  PBS_TRY(check_count(a, 2ll * a.c.kv_heads));
  return launch_paged_gather(a, kt, vt, (cudaStream_t)stream);
}

int pbs_paged_attn_workspace(const pbs_paged_cache_t* cache, const pbs_paged_batch_t* batch, int32_t q_heads, int64_t* bytes) {
  PagedArgs a;
  PBS_NONNULL(bytes);
  PBS_TRY(check_paged(cache, batch, &a));
  PBS_TRY(check_q_heads(a, q_heads));
  return paged_attn_workspace(a, q_heads, bytes);
}

int pbs_paged_attn(const pbs_paged_cache_t* cache, const pbs_paged_batch_t* batch, int32_t q_heads, const void* q, const int64_t q_strides[4],
                   void* out, const int64_t out_strides[4], float scale, void* workspace, int64_t workspace_bytes, void* stream) {
  PagedArgs a;
  RowTensor qt, ot;
  PBS_TRY(check_paged(cache, batch, &a));
  PBS_TRY(check_q_heads(a, q_heads));
  PBS_TRY(check_rows("q", a, q_heads, q, q_strides, false, &qt));
  PBS_TRY(check_rows("out", a, q_heads, out, out_strides, true, &ot));
  PBS_NONNULL(workspace);
  if ((uintptr_t)workspace % 16) { set_error("workspace: 16-byte alignment"); return PBS_ERR_LAYOUT; }
  int64_t need;
  PBS_TRY(paged_attn_workspace(a, q_heads, &need));
  if (workspace_bytes < need) { set_error("workspace: %lld bytes, need %lld", (long long)workspace_bytes, (long long)need); return PBS_ERR_SHAPE; }
  return launch_paged_attn(a, q_heads, qt, ot, scale, workspace, (cudaStream_t)stream);
}

int pbs_paged_reorder(const pbs_paged_cache_t* const* caches, int32_t layers, const pbs_paged_batch_t* batch, int32_t* block_table, int32_t beams,
                      const int32_t* parents, int64_t parents_stride, void* stream) {
  PBS_NONNULL(caches);
  PBS_NONNULL(batch);
  PBS_NONNULL(block_table);
  PBS_NONNULL(parents);
  if (layers < 1) { set_error("%d layers", layers); return PBS_ERR_SHAPE; }
  if (beams < 1 || beams > 32 || batch->batch % beams) { set_error("%d rows in groups of %d: need 1 .. 32 that divide them", batch->batch, beams); return PBS_ERR_SHAPE; }
  if (parents_stride < 0 || (batch->batch > 1 && batch->table_stride < batch->max_pages)) { set_error("rows of the block table share memory, or a negative stride"); return PBS_ERR_LAYOUT; }
  PagedArgs a;
  pbs_paged_batch_t b = *batch;
  b.block_table = block_table;
  b.new_tokens = 1;
  b.new_lens = nullptr;
  for (int32_t l = layers - 1; l >= 0; --l) {              // (the first stays in a)
    PBS_TRY(check_paged(caches[l], &b, &a));
    const pbs_paged_cache_t &c = *caches[l], &d = *caches[0];
    bool same = c.num_pages == d.num_pages && c.page_size == d.page_size && c.kv_heads == d.kv_heads && c.head_dim == d.head_dim && c.bits == d.bits;
    same = same && (c.bits != 4 || c.group_size == d.group_size) && (c.bits != 8 || c.block_size == d.block_size) && (c.bits == 16 || c.dtype == d.dtype);
    for (int i = 0; i < 3; ++i) {
      same = same && c.k_strides[i] == d.k_strides[i] && c.v_strides[i] == d.v_strides[i];
      same = same && (c.bits == 16 || (c.k_params_strides[i] == d.k_params_strides[i] && c.v_params_strides[i] == d.v_params_strides[i]));
    }
    for (int32_t m = 0; m < l; ++m)
      if (caches[m] && caches[m]->k == c.k) { set_error("layers %d and %d are one cache", m, l); return PBS_ERR_ARG; }
    if (!same) { set_error("the caches of a call have one layout: that of layer %d differs from the first's", l); return PBS_ERR_SHAPE; }
  }
  if (a.c.kv_heads > (INT_MAX >> 1)) { set_error("%d heads", a.c.kv_heads); return PBS_ERR_SHAPE; }
  return launch_paged_reorder(a, caches, layers, block_table, parents, parents_stride, beams, (cudaStream_t)stream);
}

int pbs_beam_select_workspace(const pbs_beam_select_t* args, int64_t* bytes) {
  PBS_NONNULL(bytes);
  PBS_TRY(check_beams(args));
  return beam_select_workspace(*args, bytes);
}

int pbs_beam_select(const pbs_beam_select_t* args, void* workspace, int64_t workspace_bytes, void* stream) {
  PBS_TRY(check_beams(args));
  PBS_NONNULL(workspace);
  if ((uintptr_t)workspace % 16) { set_error("workspace: 16-byte alignment"); return PBS_ERR_LAYOUT; }
  int64_t need;
  PBS_TRY(beam_select_workspace(*args, &need));
  if (workspace_bytes < need) { set_error("workspace: %lld bytes, need %lld", (long long)workspace_bytes, (long long)need); return PBS_ERR_SHAPE; }
  return launch_beam_select(*args, workspace, (cudaStream_t)stream);
}

int pbs_process_logits(const pbs_logits_t* args, void* stream) {
  PBS_NONNULL(args);
  pbs_logits_t a = *args;
  if (a.dtype < PBS_BF16 || a.dtype > PBS_FP32) { set_error("dtype %d is not bf16/fp16/fp32", a.dtype); return PBS_ERR_ARG; }
  if (a.rows < 1 || a.vocab < 1 || a.rows > 65535 || a.vocab > (1 << 30)) { set_error("logits: %d rows of %d", a.rows, a.vocab); return PBS_ERR_SHAPE; }
  PBS_NONNULL(a.logits);
  PBS_NONNULL(a.out);
  const int e = elem_bytes(a.dtype);
  if (((uintptr_t)a.logits | (uintptr_t)a.out) % e || (a.rows > 1 && (a.out_stride < a.vocab || a.logits_stride < 0))) {
    set_error("logits: rows of out must not share memory, strides must not be negative");
    return PBS_ERR_LAYOUT;
  }
  if (a.history < 0 || a.history >= (1 << 30) || a.biases < 0 || a.biases >= (1 << 30)) { set_error("logits: history %d, biases %d", a.history, a.biases); return PBS_ERR_SHAPE; }
  if (a.tokens && a.token_bytes != 4 && a.token_bytes != 8) { set_error("tokens: integers of %d bytes", a.token_bytes); return PBS_ERR_ARG; }
  if (a.history == 0) a.tokens = nullptr;
  if (a.biases == 0) a.bias_ids = nullptr;
  if (a.bias_ids) {
    PBS_NONNULL(a.bias_values);
    if (a.bias_id_bytes != 4 && a.bias_id_bytes != 8) { set_error("bias_ids: integers of %d bytes", a.bias_id_bytes); return PBS_ERR_ARG; }
  }
  return launch_process_logits(a, (cudaStream_t)stream);
}

}  // extern "C"
