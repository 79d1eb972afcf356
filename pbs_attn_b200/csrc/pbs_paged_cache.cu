// New keys and values into a paged cache, rotated and quantised on the way, and back.
//
// D / 8 neighbouring lanes hold a row of D channels, eight each: a lane's channels are 16 bytes of the input and, in 4 bits, one word of the
// cache.  The other half of a row, for the rotation, is D / 16 lanes away, and a group's extremes (4 bits) meet over G / 8 lanes, so 16 and 4 bits
// need no shared memory, and every byte is read and written once.  A CTA's groups of lanes take neighbouring tokens and the same heads, of the
// queries, the keys or the values, so nothing branches within a warp and codes of neighbouring tokens are written together.  8 bits: see below.
//
// HBM bounds prompts, latency and the launch single tokens.  8191 tokens of 8 KV heads into 4 bits: 15 us (33.5 MB read, 9.4 MB written, 2.9
// TB/s; 75 % of the issue slots are taken: some 170 instructions for eight channels), back out 8.9 us; 64 sequences' next tokens, 32 query
// heads rotated, 2.3 us.  Into 8 bits 11.2 us (50 MB, 4.5 TB/s, 68 %; 64 % of the issue slots: a warp's loads, maximum, scale and stores come one
// after another, and nothing of a next block is under way) and back 8.9 (86 %); one token 2.5 us, 64 sequences' 3.0, with drafts of up to four 3.1.
#include <climits>
#include <type_traits>

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

// A lane's eight channels of a row that LPR lanes hold, rotated: x cos + rotate_half(x) sin, each product and the sum rounded.
template <class T, int LPR>
__device__ __forceinline__ void turned8(const uint4& now, const uint4& cs, const uint4& sn, int lane, float (&x)[8]) {
  const uint4 other = make_uint4(__shfl_xor_sync(0xffffffffu, now.x, LPR / 2), __shfl_xor_sync(0xffffffffu, now.y, LPR / 2),
                                 __shfl_xor_sync(0xffffffffu, now.z, LPR / 2), __shfl_xor_sync(0xffffffffu, now.w, LPR / 2));
  float y[8], cf[8], sf[8];
  unpack8<T>(now, x);
  unpack8<T>(other, y);
  unpack8<T>(cs, cf);
  unpack8<T>(sn, sf);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = __fadd_rn(__fmul_rn(x[j], cf[j]), __fmul_rn(lane < LPR / 2 ? -y[j] : y[j], sf[j]));
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
  after_the_kernel_before();
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
    if (turn) turned8<T, LPR>(now, cs, sn, lane, x);
    else unpack8<T>(now, x);
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

// --------------------------------------------------------------------------------------------------------------------------------
// 8 bits.  A block's scale is known when all of the call's tokens in it have been looked at, so a warp takes 16 of its tokens (a head's keys or
// values) and keeps them in registers, all loads under way at once; the warps of a block of 32 or 64 tokens meet in shared memory for the
// largest magnitude.  Where the scale of a block with older tokens has grown, their codes are brought to it by the same warps.
//
// Rounding: a product and 1.5 * 2^23 in one fma leave the code, as a signed byte, in the lowest bits of the sum.

// Largest magnitude of four words of two values; a NaN stays.
__device__ __forceinline__ float most8(const uint4& w, __nv_bfloat16*) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&u[0]));
#pragma unroll
  for (int i = 1; i < 4; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&u[i])));
  return max_nan(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float most8(const uint4& w, __half*) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  __half2 m = __habs2(*reinterpret_cast<const __half2*>(&u[0]));
#pragma unroll
  for (int i = 1; i < 4; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&u[i])));
  return max_nan(__low2float(m), __high2float(m));
}

// Codes of eight values at `inv` a step.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float inv) {
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(fmaf(x[i], inv, 12582912.f));
  return make_uint2(__byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(r[4], r[5], 0x0040), __byte_perm(r[6], r[7], 0x0040), 0x5410));
}

// The numbers that four signed bytes are.
__device__ __forceinline__ void signed4(uint32_t w, float (&x)[4]) {
  w ^= 0x80808080u;                                        // 0 .. 255, the lowest byte of 2^23 + that
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7650 + i)) - 8388736.f;
}

constexpr float kLeastScale = 7.52316385e-37f;             // 2^-120: its reciprocal is an ordinary number

// Queries, rotated: group g of lanes takes a token, and p.chunk of its heads.
template <class T, int D>
__device__ __forceinline__ void turn_queries(const AppendArgs& p, int g) {
  constexpr int LPR = D / 8;
  const pbs_paged_batch_t& bt = p.a.b;
  const int lane = threadIdx.x % LPR, token = g / p.q_chunks, head0 = g % p.q_chunks * p.chunk;
  const bool active = token < bt.batch * bt.new_tokens;    // (the other lanes go along: a warp's shuffles take all of them)
  const int n = min(p.chunk, p.q_heads - head0), seq = active ? token / bt.new_tokens : 0, i = active ? token % bt.new_tokens : 0;
  int pos = active ? new_position(bt, seq, i) : -1;
  uint4 cs = make_uint4(0, 0, 0, 0), sn = cs;
  if (pos >= 0) {
    if (p.table_rows > 0 && pos >= p.table_rows) {
      paged_fault(p.a, PBS_PAGED_BAD_ROTARY);
      pos = -1;
    } else {
      const int64_t at = (p.table_rows > 0 ? pos * p.cs_s : seq * p.cs_b + i * p.cs_s) + 8 * lane;
      cs = *reinterpret_cast<const uint4*>((const T*)p.cosp + at);
      sn = *reinterpret_cast<const uint4*>((const T*)p.sinp + at);
    }
  }
  const T* in = (const T*)p.q.p + seq * p.q.st.b + head0 * p.q.st.h + i * p.q.st.s + 8 * lane;
  T* out = (T*)p.qo.p + seq * p.qo.st.b + head0 * p.qo.st.h + i * p.qo.st.s + 8 * lane;
  for (int r = 0; r < p.chunk; ++r) {
    uint4 w = r < n ? *reinterpret_cast<const uint4*>(in + r * p.q.st.h) : make_uint4(0, 0, 0, 0);
    float x[8];
    turned8<T, LPR>(w, cs, sn, lane, x);
    w = pack8<T>(x);
    if (pos < 0) w = make_uint4(0, 0, 0, 0);               // (a row that is left out)
    if (active && r < n) *reinterpret_cast<uint4*>(out + r * p.qo.st.h) = w;
  }
}

// A block of a sequence's tokens, of a head's keys or values, that new ones come into.
struct Block {
  int seq, head, shift, first, end, begin;                 // first .. end - 1: positions of its new tokens; shift: of the call's first row; begin: of the block
  bool is_v, covers;                                       // covers: there are any
};

// Unit u of the call's: heads go fastest, then keys and values, then the `blocks` that a sequence's new tokens may lie in.
__device__ __forceinline__ Block block_of(const AppendArgs& p, int u, int blocks) {
  const pbs_paged_batch_t& bt = p.a.b;
  Block b;
  b.head = u % p.a.c.kv_heads;
  int rest = u / p.a.c.kv_heads;
  b.is_v = rest % 2;
  rest /= 2;
  b.seq = rest / blocks;
  const int n = bt.new_lens ? min(max(bt.new_lens[b.seq], 0), bt.new_tokens) : bt.new_tokens, len = bt.seq_lens[b.seq];
  b.shift = len - n;
  b.end = len;
  if (p.cosp && p.table_rows > 0 && len > p.table_rows && n > 0) {
    paged_fault(p.a, PBS_PAGED_BAD_ROTARY);
    b.end = p.table_rows;
  }
  const int start = max(0, b.shift), block = (start >> p.a.block_shift) + rest % blocks;
  b.covers = n > 0 && b.end > start && block <= (b.end - 1) >> p.a.block_shift;
  b.begin = block << p.a.block_shift;
  b.first = max(start, b.begin);
  b.end = min(b.end, b.begin + p.a.c.block_size);
  return b;
}

// A block's scale with new tokens of magnitudes up to `most` in it; old: of the tokens that it holds, 0 for none.
__device__ __forceinline__ float scale_of(float most, float old) {
  const float scale = most <= 3.402823466e38f ? fmaxf(__fmul_rn(most, 1.f / 127.f), kLeastScale) : CUDART_NAN_F;
  return max_nan(scale, fabsf(old));                       // (a pool that was not filled here may have negative ones)
}

__device__ __forceinline__ uint2 scaled8(const uint2& w, float ratio) {
  float a[4], b[4], y[8];
  signed4(w.x, a);
  signed4(w.y, b);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    y[j] = a[j];
    y[j + 4] = b[j];
  }
  return codes8(y, ratio);
}

constexpr int kPrompt = 128;

// Prompts: a warp takes 16 tokens of a block, blocks of 32 and 64 are several warps'.  Four warps a CTA, ten CTAs a SM: 11.2 us for 8191 tokens, 11.1 in
// blocks of 64, 12.3 of 64 channels (eight warps, four CTAs: 11.7, 12.7 and 13.5; twelve CTAs, spilling: 14.3, 12.7 and 11.8).
template <int DT, int D, int W, bool ROPE>
__global__ void __launch_bounds__(kPrompt, D == 256 ? ROPE ? 2 : 4 : ROPE ? 4 : 10) paged_append8_kernel(const __grid_constant__ AppendArgs p, int blocks, int units) {
  after_the_kernel_before();
  using T = typename Elem<DT>::T;
  constexpr int LPR = D / 8, RPI = 32 / LPR, NI = 16 / RPI;  // lanes a row; rows at a time, and times, of a warp's 16
  const pbs_paged_cache_t& c = p.a.c;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, col = lane % LPR, unit = (int)blockIdx.x * (kPrompt / 32 / W) + warp / W;
  Block b{};
  if (unit < units) b = block_of(p, unit, blocks);
  const int t0 = b.begin + warp % W * 16 + lane / LPR;     // this lane's first token, RPI apart
  const RowTensor& src = b.is_v ? p.v : p.k;
  const T* in = (const T*)src.p + b.seq * src.st.b + b.head * src.st.h + 8 * col;
  auto fresh = [&](int k) { return b.covers && t0 + k * RPI >= b.first && t0 + k * RPI < b.end; };
  uint4 raw[NI];
#pragma unroll
  for (int k = 0; k < NI; ++k)
    raw[k] = fresh(k) ? *reinterpret_cast<const uint4*>(in + (int64_t)(t0 + k * RPI - b.shift) * src.st.s) : make_uint4(0, 0, 0, 0);
  const int page = b.covers ? page_of(p.a, b.seq, b.begin) : -1, slot = b.begin & (c.page_size - 1);
  const bool active = page >= 0, older = active && b.first > b.begin;      // older: the block holds tokens already
  float* const scale_at = (float*)(b.is_v ? c.v_params : c.k_params) +
                          (active ? slot_offset(b.is_v ? c.v_params_strides : c.k_params_strides, page, b.head, slot >> p.a.block_shift) : 0);
  const float old = older ? *scale_at : 0.f;
  float most = 0.f;
  float x[ROPE ? NI : 1][8];
  const bool turn = ROPE && !b.is_v;
  if (turn) {
#pragma unroll
    for (int k = 0; k < (ROPE ? NI : 0); ++k) {
      const int t = t0 + k * RPI;
      uint4 cs = make_uint4(0, 0, 0, 0), sn = cs;
      if (fresh(k)) {
        const int64_t at = (p.table_rows > 0 ? t * p.cs_s : b.seq * p.cs_b + (t - b.shift) * p.cs_s) + 8 * col;
        cs = *reinterpret_cast<const uint4*>((const T*)p.cosp + at);
        sn = *reinterpret_cast<const uint4*>((const T*)p.sinp + at);
      }
      turned8<T, LPR>(raw[k], cs, sn, col, x[k]);
#pragma unroll
      for (int j = 0; j < 8; ++j) most = max_nan(most, fabsf(x[k][j]));
    }
  } else {
#pragma unroll
    for (int k = 0; k < NI; ++k) most = max_nan(most, most8(raw[k], (T*)nullptr));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
  if constexpr (W > 1) {
    __shared__ float meet[kPrompt / 32];
    if (lane == 0) meet[warp] = most;
    __syncthreads();                                       // (old scales have been read, too)
    most = meet[warp / W * W];
#pragma unroll
    for (int k = 1; k < W; ++k) most = max_nan(most, meet[warp / W * W + k]);
  }
  if (!active) return;
  const float scale = scale_of(most, old), inv = __fdiv_rn(1.f, scale);
  const bool grown = older && scale != old;                // (of one that is NaN the codes are nothing)
  int8_t* const out = (int8_t*)(b.is_v ? c.v : c.k) + slot_offset(b.is_v ? c.v_strides : c.k_strides, page, b.head, 0) + 8 * col;
  const int64_t step = (b.is_v ? c.v_strides : c.k_strides)[2];
#pragma unroll
  for (int k = 0; k < NI; ++k) {
    const int t = t0 + k * RPI;
    uint2* const at = reinterpret_cast<uint2*>(out + (t & (c.page_size - 1)) * step);
    if (t >= b.first && t < b.end) {
      float y[8];
      if (turn) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = x[ROPE ? k : 0][j];
      } else {
        unpack8<T>(raw[k], y);
      }
      *at = codes8(y, inv);
    }
  }
  if (grown) {
    const float ratio = __fdiv_rn(old, scale);
#pragma unroll 1
    for (int k = 0; k < NI; ++k) {
      const int t = t0 + k * RPI;
      uint2* const at = reinterpret_cast<uint2*>(out + (t & (c.page_size - 1)) * step);
      if (t < b.first) *at = scaled8(*at, ratio);
    }
  }
  if (lane == 0 && warp % W == 0) *scale_at = scale;
}

constexpr int kFew = 4;                                    // rows of a lane

// A few tokens a sequence: a warp takes all of a block, its new tokens in registers.  Latency is all there is: lengths, then rows and the page's
// number, then the scale and what is written, in little code (with the kernel above, unrolled for 16 tokens a warp, one token took 5.2 us).
// The CTAs behind kv_ctas turn queries.
template <int DT, int D, bool ROPE>
__global__ void __launch_bounds__(kThreads) paged_append8_few_kernel(const __grid_constant__ AppendArgs p, int blocks, int units, int kv_ctas) {
  after_the_kernel_before();
  using T = typename Elem<DT>::T;
  constexpr int LPR = D / 8, RPI = 32 / LPR;
  if (ROPE && (int)blockIdx.x >= kv_ctas) {
    turn_queries<T, D>(p, ((int)blockIdx.x - kv_ctas) * (kThreads / LPR) + threadIdx.x / LPR);
    return;
  }
  const pbs_paged_cache_t& c = p.a.c;
  const int lane = threadIdx.x % 32, col = lane % LPR, unit = (int)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
  if (unit >= units) return;
  const Block b = block_of(p, unit, blocks);
  if (!b.covers) return;
  const RowTensor& src = b.is_v ? p.v : p.k;
  const T* in = (const T*)src.p + b.seq * src.st.b + b.head * src.st.h + 8 * col;
  const int t0 = b.first + lane / LPR;
  const bool turn = ROPE && !b.is_v;
  uint4 raw[kFew], cs[kFew], sn[kFew];
#pragma unroll
  for (int k = 0; k < kFew; ++k) {
    const int t = t0 + k * RPI;
    raw[k] = cs[k] = sn[k] = make_uint4(0, 0, 0, 0);
    if (t >= b.end) continue;
    raw[k] = *reinterpret_cast<const uint4*>(in + (int64_t)(t - b.shift) * src.st.s);
    if (turn) {
      const int64_t at = (p.table_rows > 0 ? t * p.cs_s : b.seq * p.cs_b + (t - b.shift) * p.cs_s) + 8 * col;
      cs[k] = *reinterpret_cast<const uint4*>((const T*)p.cosp + at);
      sn[k] = *reinterpret_cast<const uint4*>((const T*)p.sinp + at);
    }
  }
  const int page = page_of(p.a, b.seq, b.begin), slot = b.begin & (c.page_size - 1);
  if (page < 0) return;                                    // (the whole warp's)
  const bool older = b.first > b.begin;
  float* const scale_at = (float*)(b.is_v ? c.v_params : c.k_params) + slot_offset(b.is_v ? c.v_params_strides : c.k_params_strides, page, b.head, slot >> p.a.block_shift);
  const float old = older ? *scale_at : 0.f;
  float most = 0.f, x[kFew][8];
#pragma unroll
  for (int k = 0; k < kFew; ++k) {
    if (b.first + k * RPI >= b.end) break;
    if (turn) turned8<T, LPR>(raw[k], cs[k], sn[k], col, x[k]);
    else unpack8<T>(raw[k], x[k]);
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max_nan(most, fabsf(x[k][j]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
  const float scale = scale_of(most, old), inv = __fdiv_rn(1.f, scale);
  int8_t* const out = (int8_t*)(b.is_v ? c.v : c.k) + slot_offset(b.is_v ? c.v_strides : c.k_strides, page, b.head, 0) + 8 * col;
  const int64_t step = (b.is_v ? c.v_strides : c.k_strides)[2];
  auto at = [&](int t) { return reinterpret_cast<uint2*>(out + (t & (c.page_size - 1)) * step); };
#pragma unroll
  for (int k = 0; k < kFew; ++k) {
    if (b.first + k * RPI >= b.end) break;
    if (t0 + k * RPI < b.end) *at(t0 + k * RPI) = codes8(x[k], inv);
  }
  if (older && scale != old) {                             // (of one that is NaN the codes are nothing)
    const float ratio = __fdiv_rn(old, scale);
    constexpr int A = 4;                                   // rows under way
    for (int t = b.begin + lane / LPR; t < b.first; t += A * RPI) {
      uint2 w[A];
#pragma unroll
      for (int k = 0; k < A; ++k)
        if (t + k * RPI < b.first) w[k] = *at(t + k * RPI);
#pragma unroll
      for (int k = 0; k < A; ++k)
        if (t + k * RPI < b.first) *at(t + k * RPI) = scaled8(w[k], ratio);
    }
  }
  if (lane == 0) *scale_at = scale;
}

template <int DT, int D, int BITS, int G>
__global__ void __launch_bounds__(kThreads, 4) paged_gather_kernel(const __grid_constant__ AppendArgs p, int tokens) {
  after_the_kernel_before();
  using T = typename Elem<DT>::T;
  constexpr int LPR = D / 8;
  const pbs_paged_cache_t& c = p.a.c;
  const bool is_v = (int)blockIdx.y >= p.kv_chunks;
  const int head0 = ((int)blockIdx.y - (is_v ? p.kv_chunks : 0)) * p.chunk, n = min(p.chunk, c.kv_heads - head0);
  const int lane = threadIdx.x % LPR, token = blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  if (token >= tokens) return;
  const int seq = token / p.a.b.new_tokens, i = token % p.a.b.new_tokens;
  const int pos = new_position(p.a.b, seq, i);
  const int page = pos >= 0 ? page_of(p.a, seq, pos) : -1, slot = pos & (c.page_size - 1);   // (0 .. page_size - 1, of -1 too)
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
  if (BITS == 8) {
    pin = (const uint8_t*)((const float*)(is_v ? c.v_params : c.k_params) +
                           slot_offset(is_v ? c.v_params_strides : c.k_params_strides, max(page, 0), head0, slot >> p.a.block_shift));
    pstep = (is_v ? c.v_params_strides : c.k_params_strides)[1] * 4;
  }
  const RowTensor& dst = is_v ? p.v : p.k;
  T* out = (T*)dst.p + seq * dst.st.b + head0 * dst.st.h + i * dst.st.s + 8 * lane;
  const float most = finite_max((T*)nullptr);
  constexpr int U = 4;                                     // rows that a lane has under way
  for (int r = 0; r < n; r += U) {
    uint4 w[U];                                            // 4 bits: word and params in x and y; 8: codes in x and y, scale in z
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = make_uint4(0, 0, 0, 0);
      if (r + u >= n || page < 0) continue;
      if constexpr (BITS == 16) {
        w[u] = *reinterpret_cast<const uint4*>(in + u * step);
      } else if constexpr (BITS == 8) {
        const uint2 codes = *reinterpret_cast<const uint2*>(in + u * step);
        w[u] = make_uint4(codes.x, codes.y, *reinterpret_cast<const uint32_t*>(pin + u * pstep), 0);
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
      if constexpr (BITS == 8) {
        const float scale = __uint_as_float(w[u].z);
        float a[4], b[4], x[8];
        signed4(w[u].x, a);
        signed4(w[u].y, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = a[j] * scale;
          x[j + 4] = b[j] * scale;
        }
        if (127.f * fabsf(scale) > most) {                        // (a key that the rotation made larger than fp16 holds)
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = fminf(fmaxf(x[j], -most), most);
        }
        w[u] = pack8<T>(x);
        if (page < 0) w[u] = make_uint4(0, 0, 0, 0);
      }
      *reinterpret_cast<uint4*>(out + u * dst.st.h) = w[u];
    }
    in += U * step;
    pin += U * pstep;
    out += U * dst.st.h;
  }
}

// A group of lanes takes so many of a token's rows that all groups are resident at a time: what the rows of a token share (position, page,
// rotary factors, the index arithmetic) is then read and done once for them.  One token: a row each.
template <int D>
dim3 deal(AppendArgs& p) {
  constexpr int RPB = kThreads / (D / 8);
  const int64_t tokens = (int64_t)p.a.b.batch * p.a.b.new_tokens, resident = (int64_t)device_sms() * 4 * RPB;
  const int64_t chunk = (tokens * (p.q_heads + 2 * p.a.c.kv_heads) + resident - 1) / resident;
  p.chunk = (int)(chunk < 8 ? chunk : 8);
  p.q_chunks = (p.q_heads + p.chunk - 1) / p.chunk;
  p.kv_chunks = (p.a.c.kv_heads + p.chunk - 1) / p.chunk;
  return dim3((unsigned)((tokens + RPB - 1) / RPB), (unsigned)(p.q_chunks + 2 * p.kv_chunks));
}

template <int DT, int D, int BITS, int G>
int launch_gather(AppendArgs p, cudaStream_t st) {
  const dim3 grid = deal<D>(p);
  PBS_LAUNCH_EARLY("paged_gather_kernel", (paged_gather_kernel<DT, D, BITS, G>), grid, kThreads, st, p, p.a.b.batch * p.a.b.new_tokens);
  PBS_CUDA_CHECK_LAUNCH("paged_gather_kernel");
  return PBS_OK;
}

template <int DT, int D, int BITS, int G>
int launch(AppendArgs p, bool gather, cudaStream_t st) {
  if (gather) return launch_gather<DT, D, BITS, G>(p, st);
  const dim3 grid = deal<D>(p);
  PBS_LAUNCH_EARLY("paged_append_kernel", (paged_append_kernel<DT, D, BITS, G>), grid, kThreads, st, p, p.a.b.batch * p.a.b.new_tokens);
  PBS_CUDA_CHECK_LAUNCH("paged_append_kernel");
  return PBS_OK;
}

template <int DT, int D>
int launch_append8(AppendArgs p, cudaStream_t st) {
  constexpr int RPB = kThreads / (D / 8), RPI = 256 / D;
  const int S = p.a.b.new_tokens, bs = p.a.c.block_size;
  const int64_t blocks = ((int64_t)S + 2 * bs - 2) / bs;   // that S tokens reach into, wherever they begin
  const int64_t units = blocks * p.a.b.batch * 2 * p.a.c.kv_heads, tokens = (int64_t)p.a.b.batch * S;
  if (units > INT_MAX - 1024) { set_error("paged append: too many blocks of tokens in a call"); return PBS_ERR_SHAPE; }
  if (S <= kFew * RPI) {
    // heads of a token's queries share its rotary factors: as many as leave every group of lanes something to do
    const int64_t groups = (int64_t)device_sms() * 4 * RPB, chunk = (tokens * p.q_heads + groups - 1) / groups, kv_ctas = (units + kThreads / 32 - 1) / (kThreads / 32);
    p.chunk = (int)(chunk < 1 ? 1 : chunk < 8 ? chunk : 8);
    p.q_chunks = (p.q_heads + p.chunk - 1) / p.chunk;
    const unsigned ctas = (unsigned)(kv_ctas + (tokens * p.q_chunks + RPB - 1) / RPB);
    if (p.cosp) PBS_LAUNCH_EARLY("paged_append8_few_kernel", (paged_append8_few_kernel<DT, D, true>), ctas, kThreads, st, p, (int)blocks, (int)units, (int)kv_ctas);
    else PBS_LAUNCH_EARLY("paged_append8_few_kernel", (paged_append8_few_kernel<DT, D, false>), (unsigned)kv_ctas, kThreads, st, p, (int)blocks, (int)units, (int)kv_ctas);
    PBS_CUDA_CHECK_LAUNCH("paged_append8_few_kernel");
    return PBS_OK;
  }
  auto prompt = [&](auto warps) -> int {
    constexpr int W = decltype(warps)::value, UPC = kPrompt / 32 / W;
    const unsigned ctas = (unsigned)((units + UPC - 1) / UPC);
    if (p.cosp) PBS_LAUNCH_EARLY("paged_append8_kernel", (paged_append8_kernel<DT, D, W, true>), ctas, kPrompt, st, p, (int)blocks, (int)units);
    else PBS_LAUNCH_EARLY("paged_append8_kernel", (paged_append8_kernel<DT, D, W, false>), ctas, kPrompt, st, p, (int)blocks, (int)units);
    return PBS_OK;
  };
  if (bs == 16) PBS_TRY(prompt(std::integral_constant<int, 1>()));
  else if (bs == 32) PBS_TRY(prompt(std::integral_constant<int, 2>()));
  else PBS_TRY(prompt(std::integral_constant<int, 4>()));
  PBS_CUDA_CHECK_LAUNCH("paged_append8_kernel");
  if (p.q_heads) {                                         // the queries, which cost as much as keys and values, by the kernel that is made for them
    dim3 grid = deal<D>(p);
    grid.y = p.q_chunks;
    PBS_LAUNCH_EARLY("paged_append_kernel", (paged_append_kernel<DT, D, 16, 0>), grid, kThreads, st, p, (int)tokens);
    PBS_CUDA_CHECK_LAUNCH("paged_append_kernel");
  }
  return PBS_OK;
}

template <int DT, int D>
int by_bits(const AppendArgs& p, bool gather, cudaStream_t st) {
  if (p.a.c.bits == 16) return launch<DT, D, 16, 0>(p, gather, st);
  if (p.a.c.bits == 8) {
    if (gather) return launch_gather<DT, D, 8, 0>(p, st);
    return launch_append8<DT, D>(p, st);
  }
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
