// Causal attention of new tokens over a paged cache: out = softmax(scale q K^T) V with the running maximum and sum of one pass.
//
// One CTA per row (sequence, query head, new token); its warps take every fourth token, a lane D / 32 channels, and meet at the end.
#include "pbs_paged.cuh"

namespace pbs {
namespace {

constexpr int kWarps = 4;

struct AttnArgs {
  PagedArgs a;
  RowTensor q, out;
  int q_heads;
  float scale;                                             // times log2(e)
};

template <int DT, int D, int BITS>
__device__ __forceinline__ void load_row(const pbs_paged_cache_t& c, bool is_v, int page, int head, int slot, int lane, float (&x)[D / 32]) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int N = D / 32;
  if constexpr (BITS == 16) {
    const T* p = (const T*)(is_v ? c.v : c.k) + slot_offset(is_v ? c.v_strides : c.k_strides, page, head, slot) + N * lane;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = E::ld(p + j);
  } else {
    const uint8_t* p = (const uint8_t*)(is_v ? c.v : c.k) + slot_offset(is_v ? c.v_strides : c.k_strides, page, head, slot) + N / 2 * lane;
    const T* pp = (const T*)(is_v ? c.v_params : c.k_params) + slot_offset(is_v ? c.v_params_strides : c.k_params_strides, page, head, slot) +
                  2 * (N * lane / c.group_size);
    const float step = E::ld(pp), low = E::ld(pp + 1);
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = fmaf((float)((p[j / 2] >> (4 * (j % 2))) & 15), step, low);
  }
}

template <int DT, int D, int BITS>
__global__ void __launch_bounds__(32 * kWarps) paged_attn_kernel(const __grid_constant__ AttnArgs p) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int N = D / 32;
  const pbs_paged_cache_t& c = p.a.c;
  const int i = blockIdx.x % p.a.b.new_tokens, seq = blockIdx.x / p.a.b.new_tokens, qh = blockIdx.y, head = qh / (p.q_heads / c.kv_heads);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int last = new_position(p.a.b, seq, i);
  float q[N], o[N] = {}, m = -CUDART_INF_F, l = 0.f;
  const T* qp = (const T*)p.q.p + seq * p.q.st.b + qh * p.q.st.h + i * p.q.st.s + N * lane;
#pragma unroll
  for (int j = 0; j < N; ++j) q[j] = E::ld(qp + j) * p.scale;
  for (int t = warp; t <= last; t += kWarps) {
    const int page = page_of(p.a, seq, t);
    if (page < 0) {
      if ((t >> p.a.shift) >= p.a.b.max_pages) break;
      continue;
    }
    float x[N], s = 0.f;
    load_row<DT, D, BITS>(c, false, page, head, t & (c.page_size - 1), lane, x);
#pragma unroll
    for (int j = 0; j < N; ++j) s = fmaf(q[j], x[j], s);
    s = warp_sum(s);
    const float top = fmaxf(m, s), w = s == -CUDART_INF_F ? 0.f : exp2f(s - top), keep = m == -CUDART_INF_F ? 0.f : exp2f(m - top);
    load_row<DT, D, BITS>(c, true, page, head, t & (c.page_size - 1), lane, x);
    l = fmaf(l, keep, w);
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = fmaf(w, x[j], o[j] * keep);
    m = top;
  }
  __shared__ float so[kWarps][D], sm[kWarps], sl[kWarps];
#pragma unroll
  for (int j = 0; j < N; ++j) so[warp][N * lane + j] = o[j];
  if (lane == 0) { sm[warp] = m; sl[warp] = l; }
  __syncthreads();
  float top = -CUDART_INF_F, sum = 0.f;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w]);
  float wt[kWarps];
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    wt[w] = sm[w] == -CUDART_INF_F && sl[w] == 0.f ? 0.f : exp2f(sm[w] - top);
    sum = fmaf(wt[w], sl[w], sum);
  }
  for (int d = threadIdx.x; d < D; d += 32 * kWarps) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) x = fmaf(wt[w], so[w][d], x);
    ((T*)p.out.p)[seq * p.out.st.b + qh * p.out.st.h + i * p.out.st.s + d] = E::cvt(sum == 0.f ? 0.f : x / sum);
  }
}

template <int DT, int D>
int launch(const AttnArgs& p, cudaStream_t st) {
  const dim3 grid((unsigned)(p.a.b.batch * p.a.b.new_tokens), (unsigned)p.q_heads);
  if (p.a.c.bits == 16) paged_attn_kernel<DT, D, 16><<<grid, 32 * kWarps, 0, st>>>(p);
  else paged_attn_kernel<DT, D, 4><<<grid, 32 * kWarps, 0, st>>>(p);
  PBS_CUDA_CHECK_LAUNCH("paged_attn_kernel");
  return PBS_OK;
}

template <int DT>
int by_dim(const AttnArgs& p, cudaStream_t st) {
  return p.a.c.head_dim == 64 ? launch<DT, 64>(p, st) : p.a.c.head_dim == 128 ? launch<DT, 128>(p, st) : launch<DT, 256>(p, st);
}

}  // namespace

int64_t paged_attn_workspace(const PagedArgs&, int) { return PBS_PAGED_COUNTER_BYTES; }

int launch_paged_attn(const PagedArgs& a, int q_heads, const RowTensor& q, const RowTensor& out, float scale, void*, cudaStream_t st) {
  const AttnArgs p{a, q, out, q_heads, scale * 1.44269504f};
  return a.c.dtype == PBS_BF16 ? by_dim<PBS_BF16>(p, st) : by_dim<PBS_FP16>(p, st);
}

}  // namespace pbs
