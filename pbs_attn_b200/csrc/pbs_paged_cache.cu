// New keys and values into a paged cache, rotated and quantised on the way, and back.
//
// D / 8 neighbouring lanes hold a row of D channels, eight each: a lane's channels are 16 bytes of the input and, in 4 bits, one word of the
// cache.  The other half of a row, for the rotation, is D / 16 lanes away, and a group's extremes meet over G / 8 lanes, so no shared memory
// is needed and every byte is read and written once.  A CTA's groups of lanes take neighbouring tokens and the same heads, of the queries, the
// keys or the values, so nothing branches within a warp and codes of neighbouring tokens are written together.
//
// HBM bounds prompts, latency and the launch single tokens.  8191 tokens of 8 KV heads into 4 bits: 15 us (33.5 MB read, 9.4 MB written, 2.9
// TB/s; 75 % of the issue slots are taken: some 170 instructions for eight channels), back out 11 us; 64 sequences' next tokens, 32 query
// heads rotated, 2.5 us.
#include "pbs_paged.cuh"

namespace pbs {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16*) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ float2 unpack2(uint32_t w, __half*) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half*) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <class T>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2(u[i], (T*)nullptr);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

template <class T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2(x[0], x[1], (T*)nullptr), pack2(x[2], x[3], (T*)nullptr), pack2(x[4], x[5], (T*)nullptr), pack2(x[6], x[7], (T*)nullptr));
}

// Largest finite number of the type: a minimum beyond them (a key that the rotation made larger than fp16 holds) stays finite.
__device__ __forceinline__ float finite_max(__nv_bfloat16*) { return 3.38953139e38f; }
__device__ __forceinline__ float finite_max(__half*) { return 65504.f; }

__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Codes of a lane's eight channels of a group that LANES lanes share; params: step (low half) and minimum (high half).
template <class T, int LANES>
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t& params) {
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const float most = finite_max((T*)nullptr);
  // halves first: the range of two large numbers of opposite sign is not representable
  const float range = __fsub_rn(hi * 0.5f, lo * 0.5f);
  params = range <= 3.402823466e38f ? pack2(__fmul_rn(range, 2.f / 15.f), fminf(fmaxf(lo, -most), most), (T*)nullptr)
                                    : pack2(0.f, CUDART_NAN_F, (T*)nullptr);       // (an infinity or a NaN in the group)
  const float2 p = unpack2(params, (T*)nullptr);
  const float inv = p.x > 0.f ? __fdiv_rn(1.f, p.x) : 0.f;
  // rounded by adding 1.5 * 2^23, whose sums have the code in their lowest bits; eight of them, four bits apart, less what 1.5 * 2^23 itself
  // sums up to.  (A conversion and a rounding instruction each took four times as long.)
  constexpr float kRound = 12582912.f;
  constexpr uint32_t kBits = 0x4b400000u;
  uint32_t word = 0, excess = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) excess += kBits << 4 * i;
  const float least_code = __fmul_rn(__fsub_rn(lo, p.y), inv), most_code = __fmul_rn(__fsub_rn(hi, p.y), inv);
  if (least_code >= -0.5f && most_code < 15.5f) {          // (the extremes round to 0 .. 15, and all between them)
#pragma unroll
    for (int i = 0; i < 8; ++i) word += __float_as_uint(__fadd_rn(__fmul_rn(__fsub_rn(x[i], p.y), inv), kRound)) << 4 * i;
  } else {                                                 // step and minimum were rounded by more than a code
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // a step below the smallest normal number has an infinite reciprocal; its product with 0 is NaN, which fmaxf takes for 0
      const float c = fminf(fmaxf(__fmul_rn(__fsub_rn(x[i], p.y), inv), 0.f), 15.f);
      word += __float_as_uint(__fadd_rn(c, kRound)) << 4 * i;
    }
  }
  return word - excess;
}

struct AppendArgs {
  PagedArgs a;
  RowTensor k, v, q, qo;
  const void* cosp;
  const void* sinp;
  int64_t cs_b, cs_s;
  int q_heads, table_rows;
  int chunk, q_chunks, kv_chunks;                          // rows of a token that a group of lanes takes; pieces that queries, keys, values come to
};

constexpr int kAhead = 2;                                  // rows that a lane has under way

template <int DT, int D, int BITS, int G>
__global__ void __launch_bounds__(kThreads, 4) paged_append_kernel(const __grid_constant__ AppendArgs p, int tokens) {
  using T = typename Elem<DT>::T;
  constexpr int LPR = D / 8;                               // lanes a row
  const pbs_paged_cache_t& c = p.a.c;
  // what this CTA's rows are: heads head .. head + n - 1 of the queries, keys or values of neighbouring tokens, a token a group of lanes
  const int piece = blockIdx.y;
  const bool is_q = piece < p.q_chunks, is_v = piece >= p.q_chunks + p.kv_chunks;
  const int head0 = (is_q ? piece : is_v ? piece - p.q_chunks - p.kv_chunks : piece - p.q_chunks) * p.chunk;
  const int n = min(p.chunk, (is_q ? p.q_heads : c.kv_heads) - head0);
  const RowTensor& src = is_q ? p.q : is_v ? p.v : p.k;
  const int lane = threadIdx.x % LPR, token = blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  const bool active = token < tokens;                      // (the other lanes go along: a warp's shuffles take all of them)
  const int seq = active ? token / p.a.b.new_tokens : 0, i = active ? token % p.a.b.new_tokens : 0;
  const T* in = (const T*)src.p + seq * src.st.b + head0 * src.st.h + i * src.st.s + 8 * lane;
  const int64_t step = src.st.h;
  uint4 raw[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    if (u < n) raw[u] = *reinterpret_cast<const uint4*>(in + u * step);
  int pos = active ? new_position(p.a.b, seq, i) : -1;
  const bool turn = p.cosp && !is_v;
  uint4 cs = make_uint4(0, 0, 0, 0), sn = cs;
  if (p.cosp && pos >= 0) {
    if (p.table_rows > 0 && pos >= p.table_rows) {
      paged_fault(p.a, PBS_PAGED_BAD_ROTARY);
      pos = -1;
    } else if (turn) {
      const int64_t at = (p.table_rows > 0 ? pos * p.cs_s : seq * p.cs_b + i * p.cs_s) + 8 * lane;
      cs = *reinterpret_cast<const uint4*>((const T*)p.cosp + at);
      sn = *reinterpret_cast<const uint4*>((const T*)p.sinp + at);
    }
  }
  const int page = pos >= 0 && !is_q ? page_of(p.a, seq, pos) : -1, slot = pos & (c.page_size - 1);
  const bool writes = is_q ? active : page >= 0;
  // where the rows go, and their params, from head to head
  uint8_t *out, *pout = nullptr;
  int64_t out_step, pout_step = 0;
  if (is_q) {
    out = (uint8_t*)((T*)p.qo.p + seq * p.qo.st.b + head0 * p.qo.st.h + i * p.qo.st.s + 8 * lane);
    out_step = p.qo.st.h * (int)sizeof(T);
  } else {
    constexpr int ES = BITS == 16 ? 2 : 1;
    out = (uint8_t*)(is_v ? c.v : c.k) + slot_offset(is_v ? c.v_strides : c.k_strides, max(page, 0), head0, slot) * ES + lane * BITS;
    out_step = (is_v ? c.v_strides : c.k_strides)[1] * ES;
    if (BITS == 4) {
      pout = (uint8_t*)((T*)(is_v ? c.v_params : c.k_params) + slot_offset(is_v ? c.v_params_strides : c.k_params_strides, max(page, 0), head0, slot)) +
             lane / (G / 8) * 4;
      pout_step = (is_v ? c.v_params_strides : c.k_params_strides)[1] * (int)sizeof(T);
    }
  }
  for (int r = 0; r < n; ++r) {
    const uint4 now = raw[0];
#pragma unroll
    for (int u = 0; u + 1 < kAhead; ++u) raw[u] = raw[u + 1];
    if (r + kAhead < n) raw[kAhead - 1] = *reinterpret_cast<const uint4*>(in + kAhead * step);
    in += step;
    float x[8];
    unpack8<T>(now, x);
    if (turn) {
      const uint4 other = make_uint4(__shfl_xor_sync(0xffffffffu, now.x, LPR / 2), __shfl_xor_sync(0xffffffffu, now.y, LPR / 2),
                                     __shfl_xor_sync(0xffffffffu, now.z, LPR / 2), __shfl_xor_sync(0xffffffffu, now.w, LPR / 2));
      float y[8], cf[8], sf[8];
      unpack8<T>(other, y);
      unpack8<T>(cs, cf);
      unpack8<T>(sn, sf);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __fadd_rn(__fmul_rn(x[j], cf[j]), __fmul_rn(lane < LPR / 2 ? -y[j] : y[j], sf[j]));
    }
    if (BITS == 16 || is_q) {
      uint4 w = pack8<T>(x);
      if (pos < 0) w = make_uint4(0, 0, 0, 0);             // (a query's row that is left out)
      if (writes) *reinterpret_cast<uint4*>(out) = w;
    } else {
      uint32_t params;
      const uint32_t word = quantise8<T, BITS == 4 ? G / 8 : 1>(x, params);
      if (writes) {
        *reinterpret_cast<uint32_t*>(out) = word;
        if (lane % (BITS == 4 ? G / 8 : 1) == 0) *reinterpret_cast<uint32_t*>(pout) = params;
      }
      pout += pout_step;
    }
    out += out_step;
  }
}

template <int DT, int D, int BITS, int G>
__global__ void __launch_bounds__(kThreads, 4) paged_gather_kernel(const __grid_constant__ AppendArgs p, int tokens) {
  using T = typename Elem<DT>::T;
  constexpr int LPR = D / 8;
  const pbs_paged_cache_t& c = p.a.c;
  const bool is_v = (int)blockIdx.y >= p.kv_chunks;
  const int head0 = ((int)blockIdx.y - (is_v ? p.kv_chunks : 0)) * p.chunk, n = min(p.chunk, c.kv_heads - head0);
  const int lane = threadIdx.x % LPR, token = blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  if (token >= tokens) return;
  const int seq = token / p.a.b.new_tokens, i = token % p.a.b.new_tokens;
  const int pos = new_position(p.a.b, seq, i);
  const int page = pos >= 0 ? page_of(p.a, seq, pos) : -1, slot = pos & (c.page_size - 1);
  constexpr int ES = BITS == 16 ? 2 : 1;
  const uint8_t* in = (const uint8_t*)(is_v ? c.v : c.k) + slot_offset(is_v ? c.v_strides : c.k_strides, max(page, 0), head0, slot) * ES + lane * BITS;
  const int64_t step = (is_v ? c.v_strides : c.k_strides)[1] * ES;
  const uint8_t* pin = nullptr;
  int64_t pstep = 0;
  if (BITS == 4) {
    pin = (const uint8_t*)((const T*)(is_v ? c.v_params : c.k_params) + slot_offset(is_v ? c.v_params_strides : c.k_params_strides, max(page, 0), head0, slot)) +
          lane / (BITS == 4 ? G / 8 : 1) * 4;
    pstep = (is_v ? c.v_params_strides : c.k_params_strides)[1] * (int)sizeof(T);
  }
  const RowTensor& dst = is_v ? p.v : p.k;
  T* out = (T*)dst.p + seq * dst.st.b + head0 * dst.st.h + i * dst.st.s + 8 * lane;
  const float most = finite_max((T*)nullptr);
  constexpr int U = 4;                                     // rows that a lane has under way
  for (int r = 0; r < n; r += U) {
    uint4 w[U];                                            // 4 bits: word and params in x and y
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = make_uint4(0, 0, 0, 0);
      if (r + u >= n || page < 0) continue;
      if constexpr (BITS == 16) {
        w[u] = *reinterpret_cast<const uint4*>(in + u * step);
      } else {
        w[u].x = *reinterpret_cast<const uint32_t*>(in + u * step);
        w[u].y = *reinterpret_cast<const uint32_t*>(pin + u * pstep);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r + u >= n) break;
      if constexpr (BITS == 4) {
        const float2 f = unpack2(w[u].y, (T*)nullptr);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          // the code in the lowest bits of 2^23 is 2^23 + code; code * step alone is exact
          x[j] = fmaf(__uint_as_float(0x4b000000u | (w[u].x >> 4 * j & 15)) - 8388608.f, f.x, f.y);
        }
        if (fmaf(15.f, f.x, f.y) > most) {                 // a step that was rounded up can lead past the type
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = fminf(x[j], most);
        }
        w[u] = pack8<T>(x);
      }
      *reinterpret_cast<uint4*>(out + u * dst.st.h) = w[u];
    }
    in += U * step;
    pin += U * pstep;
    out += U * dst.st.h;
  }
}

template <int DT, int D, int BITS, int G>
int launch(AppendArgs p, bool gather, cudaStream_t st) {
  // A group of lanes takes so many of a token's rows that all groups are resident at a time: what the rows of a token share (position, page,
  // rotary factors, the index arithmetic) is then read and done once for them.  One token: a row each.
  constexpr int RPB = kThreads / (D / 8);
  const int64_t tokens = (int64_t)p.a.b.batch * p.a.b.new_tokens, resident = (int64_t)device_sms() * 4 * RPB;
  const int64_t chunk = (tokens * (p.q_heads + 2 * p.a.c.kv_heads) + resident - 1) / resident;
  p.chunk = (int)(chunk < 8 ? chunk : 8);
  p.q_chunks = (p.q_heads + p.chunk - 1) / p.chunk;
  p.kv_chunks = (p.a.c.kv_heads + p.chunk - 1) / p.chunk;
  const dim3 grid((unsigned)((tokens + RPB - 1) / RPB), (unsigned)(p.q_chunks + 2 * p.kv_chunks));
  if (gather) paged_gather_kernel<DT, D, BITS, G><<<grid, kThreads, 0, st>>>(p, (int)tokens);
  else paged_append_kernel<DT, D, BITS, G><<<grid, kThreads, 0, st>>>(p, (int)tokens);
  PBS_CUDA_CHECK_LAUNCH(gather ? "paged_gather_kernel" : "paged_append_kernel");
  return PBS_OK;
}

template <int DT, int D>
int by_bits(const AppendArgs& p, bool gather, cudaStream_t st) {
  if (p.a.c.bits == 16) return launch<DT, D, 16, 0>(p, gather, st);
  return p.a.c.group_size == 32 ? launch<DT, D, 4, 32>(p, gather, st) : launch<DT, D, 4, 64>(p, gather, st);
}

template <int DT>
int by_dim(const AppendArgs& p, bool gather, cudaStream_t st) {
  return p.a.c.head_dim == 64 ? by_bits<DT, 64>(p, gather, st) : p.a.c.head_dim == 128 ? by_bits<DT, 128>(p, gather, st) : by_bits<DT, 256>(p, gather, st);
}

int by_type(const AppendArgs& p, bool gather, cudaStream_t st) {
  return p.a.c.dtype == PBS_BF16 ? by_dim<PBS_BF16>(p, gather, st) : by_dim<PBS_FP16>(p, gather, st);
}

}  // namespace

int launch_paged_append(const PagedArgs& a, const RowTensor& k, const RowTensor& v, int q_heads, const RowTensor& q, const RowTensor& qo,
                        const void* cosp, const void* sinp, int64_t cs_b, int64_t cs_s, int table_rows, cudaStream_t st) {
  return by_type(AppendArgs{a, k, v, q, qo, cosp, sinp, cs_b, cs_s, q_heads, table_rows, 0, 0, 0}, false, st);
}

int launch_paged_gather(const PagedArgs& a, const RowTensor& k, const RowTensor& v, cudaStream_t st) {
  return by_type(AppendArgs{a, k, v, {}, {}, nullptr, nullptr, 0, 0, 0, 0, 0, 0, 0}, true, st);
}

}  // namespace pbs
