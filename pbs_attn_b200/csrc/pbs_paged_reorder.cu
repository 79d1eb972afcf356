// Rows of a batch go on from other rows of their group, in the caches of all layers: a beam that is continued twice, or not at all.
//
// Full pages are shared: a row takes over its parent's entries of the block table.  The page under way is the row's own and takes the tokens
// that the parent's holds.  Groups change in place, so a thread takes the same piece of a page (or column of the table) for all rows of a
// group, reads what it needs of the rows that are continued, and only then writes: no buffer, no barrier, no order among threads.
//
// Bound by HBM: what moves is read once and written once.  One launch for up to kLayers layers; a CTA takes a group's keys or values of one head
// in some of them, and looks up once what moves.  32 layers of 8 KV heads of 128, pages of 64 tokens half full, half of the rows moving: 8 groups of
// four in 16 bits 25.7 us for 134 MB (80 % of the copy rate), 32 of eight 156 us; one of four in 8 bits 4.6 us.  (Divisions by the units of a page and
// four rows' pieces in registers whatever the number that moves, one CTA a SM: 65 us.  72 registers, three CTAs a SM, each taking twice as much:
// 27.6, 166 and 7.0; 48 registers, five: 32, 156 and 6.3.)  A group's table is one CTA's, 256 columns at a time: four rows of 1024 full pages 6.0 us, of
// 2048 8.3, of 8192 (131072 tokens in pages of 16) 21.4.
#include <climits>

#include "pbs_paged.cuh"

namespace pbs {
namespace {

constexpr int kThreads = 256;
constexpr int kLayers = 64;
constexpr int kMaxBeams = 32;

struct Pools {
  uint8_t *k, *v, *k_params, *v_params;
};

struct ReorderArgs {
  PagedArgs a;
  int32_t* table;
  const int32_t* beams;
  int64_t beams_stride;
  int n;                                  // rows of a group
  int layers, layers_cta;
  int piece_shift, word_shift;            // of a token's row, as powers of two: 16-byte pieces; 4-byte words of params (4 bits)
  Pools pools[kLayers];
};

// A row that takes something over.
struct Move {
  int row, parent, to, from, fill, full;  // rows of the batch; pages under way (-1: nothing to copy) and their tokens; full pages
};

// Brings units of a page, for all moves, from the parents' pages: per_layer of them at most in each of `layers`, units[m] of move m.  at(layer, u) is
// where unit u lies in page 0.  M: the most moves; U units are under way in a thread.
template <class UNIT, int M, int U, class F>
__device__ __forceinline__ void copy(const Move* moves, int count, int layers, int per_layer, int64_t page_bytes, F at, const int* units) {
  const float inverse = 1.f / (float)per_layer;
  const int total = layers * per_layer;
  for (int i0 = threadIdx.x; i0 < total; i0 += U * kThreads) {
    UNIT v[U][M];
    uint8_t* where[U];
    int unit[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kThreads;
      int layer = (int)((float)i * inverse);               // (of up to 2^21 units: off by one at most)
      layer += (i >= (layer + 1) * per_layer) - (i < layer * per_layer);
      unit[u] = i < total ? i - layer * per_layer : INT_MAX;
      where[u] = i < total ? at(layer, unit[u]) : nullptr;
#pragma unroll
      for (int m = 0; m < M; ++m)
        if (m < count && unit[u] < units[m]) v[u][m] = *reinterpret_cast<const UNIT*>(where[u] + moves[m].from * page_bytes);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < M; ++m)
        if (m < count && unit[u] < units[m]) *reinterpret_cast<UNIT*>(where[u] + moves[m].to * page_bytes) = v[u][m];
  }
}

template <int MAXN>
__global__ void __launch_bounds__(kThreads, MAXN == 8 ? 4 : 1) paged_reorder_kernel(const __grid_constant__ ReorderArgs p) {
  after_the_kernel_before();
  const pbs_paged_cache_t& c = p.a.c;
  const int head = blockIdx.x >> 1, is_v = blockIdx.x & 1, group = blockIdx.y, tid = threadIdx.x;
  const int layer0 = blockIdx.z * p.layers_cta, layers = min(p.layers_cta, p.layers - layer0);
  __shared__ Move moves[kMaxBeams];
  __shared__ int pieces[kMaxBeams], words[kMaxBeams];      // of a page under way, by move
  __shared__ int count, most_pieces, most_words;
  if (tid < 32) {
    const bool row = tid < p.n;
    const int seq = group * p.n + (row ? tid : 0);
    const int len = row ? p.a.b.seq_lens[seq] : 0;
    int parent = row ? p.beams[group * p.beams_stride + tid] : tid;
    const int theirs = __shfl_sync(0xffffffffu, len, parent & 31);
    if (row && ((unsigned)parent >= (unsigned)p.n || theirs != len)) {
      paged_fault(p.a, PBS_PAGED_BAD_BEAM);
      parent = tid;
    }
    Move m{seq, group * p.n + parent, -1, -1, len & (c.page_size - 1), min(max(len, 0) >> p.a.shift, p.a.b.max_pages)};
    bool moves_ = row && parent != tid && len > 0;
    if (moves_ && m.fill) {
      m.to = page_of(p.a, m.row, len);
      m.from = page_of(p.a, m.parent, len);
      moves_ = m.to >= 0 && m.from >= 0;
    }
    const uint32_t all = __ballot_sync(0xffffffffu, moves_);
    const int at = __popc(all & ((1u << tid) - 1));
    const int n_pieces = moves_ && m.fill && m.to != m.from ? m.fill << p.piece_shift : 0;
    const int n_words = n_pieces == 0 || c.bits == 16 ? 0 : c.bits == 8 ? (m.fill + c.block_size - 1) >> p.a.block_shift : m.fill << p.word_shift;
    if (moves_) {
      moves[at] = m;
      pieces[at] = n_pieces;
      words[at] = n_words;
    }
    const int wide = __reduce_max_sync(0xffffffffu, n_pieces), wide_words = __reduce_max_sync(0xffffffffu, n_words);
    if (tid == 0) {
      count = __popc(all);
      most_pieces = wide;
      most_words = wide_words;
    }
  }
  __syncthreads();
  const int n = count;
  if (n == 0) return;
  if (p.table && blockIdx.x == 0 && blockIdx.z == 0) {     // the table's full pages
    int full = 0;
    for (int m = 0; m < n; ++m) full = max(full, moves[m].full);
    for (int j = tid; j < full; j += kThreads) {
      int v[MAXN];
#pragma unroll
      for (int m = 0; m < MAXN; ++m)
        if (m < n && j < moves[m].full) v[m] = p.table[moves[m].parent * p.a.b.table_stride + j];
#pragma unroll
      for (int m = 0; m < MAXN; ++m)
        if (m < n && j < moves[m].full) p.table[moves[m].row * p.a.b.table_stride + j] = v[m];
    }
  }
  const int es = c.bits == 16 ? 2 : 1;
  const int64_t(&st)[3] = is_v ? c.v_strides : c.k_strides;
  const int64_t(&pst)[3] = is_v ? c.v_params_strides : c.k_params_strides;
  const Pools* const pools = p.pools + layer0;
  if (most_pieces) {
    auto at = [&](int layer, int u) {
      return (is_v ? pools[layer].v : pools[layer].k) + (head * st[1] + (u >> p.piece_shift) * st[2]) * es + (u & ((1 << p.piece_shift) - 1)) * 16;
    };
    const int64_t page = st[0] * es;
    // eight pieces under way in a thread, however many rows they are of
    if (n <= 2) copy<uint4, 2, 4>(moves, n, layers, most_pieces, page, at, pieces);
    else if (n <= 4) copy<uint4, 4, 2>(moves, n, layers, most_pieces, page, at, pieces);
    else copy<uint4, MAXN, 1>(moves, n, layers, most_pieces, page, at, pieces);
  }
  const int ps = c.bits == 8 ? 4 : 2;
  if (most_words)
    copy<uint32_t, MAXN, 1>(moves, n, layers, most_words, pst[0] * ps, [&](int layer, int u) {
      return (is_v ? pools[layer].v_params : pools[layer].k_params) + (head * pst[1] + (u >> p.word_shift) * pst[2]) * ps + (u & ((1 << p.word_shift) - 1)) * 4;
    }, words);
}

template <int MAXN>
int launch(const ReorderArgs& p, int groups, cudaStream_t st) {
  PBS_LAUNCH_EARLY("paged_reorder_kernel", paged_reorder_kernel<MAXN>, dim3(2 * p.a.c.kv_heads, groups, (p.layers + p.layers_cta - 1) / p.layers_cta), kThreads, st, p);
  PBS_CUDA_CHECK_LAUNCH("paged_reorder_kernel");
  return PBS_OK;
}

}  // namespace

int launch_paged_reorder(const PagedArgs& a, const pbs_paged_cache_t* const* caches, int layers, int32_t* table, const int32_t* beams, int64_t beams_stride, int n,
                         cudaStream_t st) {
  ReorderArgs p{};
  p.a = a;
  p.table = table;
  p.beams = beams;
  p.beams_stride = beams_stride;
  p.n = n;
  while (128 << p.piece_shift < a.c.head_dim * a.c.bits) ++p.piece_shift;
  while (a.c.bits == 4 && a.c.group_size << p.word_shift < a.c.head_dim) ++p.word_shift;
  const int groups = a.b.batch / n;
  for (int l0 = 0; l0 < layers; l0 += kLayers) {
    p.layers = layers - l0 < kLayers ? layers - l0 : kLayers;
    for (int l = 0; l < p.layers; ++l) {
      const pbs_paged_cache_t& c = *caches[l0 + l];
      p.pools[l] = Pools{(uint8_t*)c.k, (uint8_t*)c.v, (uint8_t*)c.k_params, (uint8_t*)c.v_params};
    }
    // as many CTAs as it takes to fill the SMs some times over (four of the common kind run on each at a time)
    const int64_t ctas = (int64_t)p.layers * groups * 2 * a.c.kv_heads, fill = (int64_t)device_sms() * 16;
    p.layers_cta = (int)((ctas + fill - 1) / fill);
    if (p.layers_cta > p.layers) p.layers_cta = p.layers;
    PBS_TRY(n <= 8 ? launch<8>(p, groups, st) : n <= 16 ? launch<16>(p, groups, st) : launch<kMaxBeams>(p, groups, st));
    p.table = nullptr;                                     // (its full pages have been seen to)
  }
  return PBS_OK;
}

}  // namespace pbs
