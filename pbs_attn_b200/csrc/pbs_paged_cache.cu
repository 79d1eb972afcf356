// New keys and values into a paged cache, rotated and quantised on the way, and back.
//
// D / 8 neighbouring lanes hold a row of D channels, eight each: a lane's channels are 16 bytes of the input and, in 4 bits, one word of the
// cache.  The other half of a row, for the rotation, is D / 16 lanes away, and a group's extremes meet over G / 8 lanes, so no shared memory
// is needed and every byte is read and written once.
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

// Codes of a lane's eight channels of a group that LANES lanes share; params: step (low half) and minimum (high half).
template <class T, int LANES>
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t& params) {
  float lo = x[0], hi = x[0];
  bool fine = fabsf(x[0]) <= 3.402823466e38f;
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    fine = fine && fabsf(x[i]) <= 3.402823466e38f;       // (false for NaN)
  }
  if (!fine) hi = CUDART_INF_F;                          // fmaxf drops NaNs: the group is told of them this way
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (hi == CUDART_INF_F) {
    params = pack2(0.f, CUDART_NAN_F, (T*)nullptr);
    return 0;
  }
  const float most = finite_max((T*)nullptr);
  // halves first: the range of two large numbers of opposite sign is not representable
  params = pack2(__fmul_rn(__fsub_rn(hi * 0.5f, lo * 0.5f), 2.f / 15.f), fminf(fmaxf(lo, -most), most), (T*)nullptr);
  const float2 p = unpack2(params, (T*)nullptr);
  const float inv = p.x > 0.f ? __fdiv_rn(1.f, p.x) : 0.f;
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // a step below the smallest normal number has an infinite reciprocal; its product with 0 is NaN, which fmaxf takes for 0
    const float c = fminf(fmaxf(rintf(__fmul_rn(__fsub_rn(x[i], p.y), inv)), 0.f), 15.f);
    word |= (uint32_t)c << (4 * i);
  }
  return word;
}

struct AppendArgs {
  PagedArgs a;
  RowTensor k, v, q, qo;
  const void* cosp;
  const void* sinp;
  int64_t cs_b, cs_s;
  int q_heads, table_rows;
};

template <int DT, int D, int BITS, int G>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const __grid_constant__ AppendArgs p, int rows) {
  using T = typename Elem<DT>::T;
  constexpr int LPR = D / 8;                               // lanes a row
  const int lane = threadIdx.x % LPR;
  const int row = blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  // row -> (sequence, new token, head): queries' heads, then keys', then values'
  const pbs_paged_cache_t& c = p.a.c;
  const int heads = p.q_heads + 2 * c.kv_heads;
  const bool active = row < rows;
  const int token = active ? row / heads : 0;
  int head = active ? row % heads : 0;
  const int seq = token / p.a.b.new_tokens, i = token % p.a.b.new_tokens;
  const RowTensor& in = head < p.q_heads ? p.q : head < p.q_heads + c.kv_heads ? p.k : p.v;
  const bool is_q = head < p.q_heads, is_v = head >= p.q_heads + c.kv_heads;
  if (!is_q) head -= is_v ? p.q_heads + c.kv_heads : p.q_heads;
  const uint4 raw = *reinterpret_cast<const uint4*>((const T*)in.p + seq * in.st.b + head * in.st.h + i * in.st.s + 8 * lane);
  int pos = active ? new_position(p.a.b, seq, i) : -1;
  float x[8];
  unpack8<T>(raw, x);
  if (p.cosp) {
    uint4 other;
    other.x = __shfl_xor_sync(0xffffffffu, raw.x, LPR / 2);
    other.y = __shfl_xor_sync(0xffffffffu, raw.y, LPR / 2);
    other.z = __shfl_xor_sync(0xffffffffu, raw.z, LPR / 2);
    other.w = __shfl_xor_sync(0xffffffffu, raw.w, LPR / 2);
    if (!is_v && pos >= 0) {
      if (p.table_rows > 0 && pos >= p.table_rows) {
        paged_fault(p.a, PBS_PAGED_BAD_ROTARY);
        pos = -1;
      } else {
        const int64_t at = (p.table_rows > 0 ? pos * p.cs_s : seq * p.cs_b + i * p.cs_s) + 8 * lane;
        float y[8], cs[8], sn[8];
        unpack8<T>(other, y);
        unpack8<T>(*reinterpret_cast<const uint4*>((const T*)p.cosp + at), cs);
        unpack8<T>(*reinterpret_cast<const uint4*>((const T*)p.sinp + at), sn);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __fadd_rn(__fmul_rn(x[j], cs[j]), __fmul_rn(lane < LPR / 2 ? -y[j] : y[j], sn[j]));
      }
    }
  }
  if (is_q) {
    uint4 w = pack8<T>(x);
    if (pos < 0) w = make_uint4(0, 0, 0, 0);
    if (active) *reinterpret_cast<uint4*>((T*)p.qo.p + seq * p.qo.st.b + head * p.qo.st.h + i * p.qo.st.s + 8 * lane) = w;
  }
  if constexpr (BITS == 16) {
    if (is_q || pos < 0) return;
    const int page = page_of(p.a, seq, pos), slot = pos & (c.page_size - 1);
    if (page < 0) return;
    T* at = (T*)(is_v ? c.v : c.k) + slot_offset(is_v ? c.v_strides : c.k_strides, page, head, slot);
    *reinterpret_cast<uint4*>(at + 8 * lane) = pack8<T>(x);
  } else {
    uint32_t params;                                       // (all lanes take part: a warp may hold rows of queries and of keys)
    const uint32_t word = quantise8<T, G / 8>(x, params);
    if (is_q || pos < 0) return;
    const int page = page_of(p.a, seq, pos), slot = pos & (c.page_size - 1);
    if (page < 0) return;
    uint8_t* at = (uint8_t*)(is_v ? c.v : c.k) + slot_offset(is_v ? c.v_strides : c.k_strides, page, head, slot);
    *reinterpret_cast<uint32_t*>(at + 4 * lane) = word;
    if (lane % (G / 8) == 0) {
      T* pp = (T*)(is_v ? c.v_params : c.k_params) + slot_offset(is_v ? c.v_params_strides : c.k_params_strides, page, head, slot);
      *reinterpret_cast<uint32_t*>(pp + 2 * (lane / (G / 8))) = params;
    }
  }
}

template <int DT, int D, int BITS, int G>
__global__ void __launch_bounds__(kThreads) paged_gather_kernel(const __grid_constant__ AppendArgs p, int rows) {
  using T = typename Elem<DT>::T;
  constexpr int LPR = D / 8;
  const int lane = threadIdx.x % LPR;
  const int row = blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  if (row >= rows) return;
  const pbs_paged_cache_t& c = p.a.c;
  const int token = row / (2 * c.kv_heads);
  int head = row % (2 * c.kv_heads);
  const bool is_v = head >= c.kv_heads;
  if (is_v) head -= c.kv_heads;
  const int seq = token / p.a.b.new_tokens, i = token % p.a.b.new_tokens;
  const int pos = new_position(p.a.b, seq, i);
  const int page = pos >= 0 ? page_of(p.a, seq, pos) : -1, slot = pos & (c.page_size - 1);
  uint4 w = make_uint4(0, 0, 0, 0);
  if (page >= 0) {
    if constexpr (BITS == 16) {
      w = *reinterpret_cast<const uint4*>((const T*)(is_v ? c.v : c.k) + slot_offset(is_v ? c.v_strides : c.k_strides, page, head, slot) + 8 * lane);
    } else {
      const uint8_t* at = (const uint8_t*)(is_v ? c.v : c.k) + slot_offset(is_v ? c.v_strides : c.k_strides, page, head, slot);
      const T* pp = (const T*)(is_v ? c.v_params : c.k_params) + slot_offset(is_v ? c.v_params_strides : c.k_params_strides, page, head, slot);
      const uint32_t word = *reinterpret_cast<const uint32_t*>(at + 4 * lane);
      const float2 f = unpack2(*reinterpret_cast<const uint32_t*>(pp + 2 * (lane / (G / 8))), (T*)nullptr);
      const float most = finite_max((T*)nullptr);
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = fmaf((float)((word >> (4 * j)) & 15), f.x, f.y);          // (the product alone is exact)
        x[j] = x[j] > most ? most : x[j] < -most ? -most : x[j];         // a step that was rounded up can lead past the type; NaN stays
      }
      w = pack8<T>(x);
    }
  }
  const RowTensor& out = is_v ? p.v : p.k;
  *reinterpret_cast<uint4*>((T*)out.p + seq * out.st.b + head * out.st.h + i * out.st.s + 8 * lane) = w;
}

template <int DT, int D, int BITS, int G>
int launch(const AppendArgs& p, bool gather, cudaStream_t st) {
  const int64_t rows = (int64_t)p.a.b.batch * p.a.b.new_tokens * (p.q_heads + 2 * p.a.c.kv_heads);
  constexpr int RPB = kThreads / (D / 8);
  const unsigned grid = (unsigned)((rows + RPB - 1) / RPB);
  if (gather) paged_gather_kernel<DT, D, BITS, G><<<grid, kThreads, 0, st>>>(p, (int)rows);
  else paged_append_kernel<DT, D, BITS, G><<<grid, kThreads, 0, st>>>(p, (int)rows);
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
  return by_type(AppendArgs{a, k, v, q, qo, cosp, sinp, cs_b, cs_s, q_heads, table_rows}, false, st);
}

int launch_paged_gather(const PagedArgs& a, const RowTensor& k, const RowTensor& v, cudaStream_t st) {
  return by_type(AppendArgs{a, k, v, {}, {}, nullptr, nullptr, 0, 0, 0, 0}, true, st);
}

}  // namespace pbs
