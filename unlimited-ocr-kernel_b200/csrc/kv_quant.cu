// kv_quant.cu — a KV cache held in 4 or 8 bits: quantised as it is written
// (a prompt's rows, or one token of every sequence, with or without its
// rotation), read back, and attended to by one query per sequence.  Layout:
// kv_quant.cuh.
//
// Per group of 32 dims of one head of one token, L = 2^bits - 1:
//   m = the largest bf16 <= min x,  s = the smallest bf16 >= (max x - m) / L,
//   code = clamp(rint((x - m) / s), 0, L)   (0 where s = 0),
// with the differences and quotients in double, rounded half to even; the
// cache stands for m + s * code.  m and s are rounded outwards so that the
// codes reach every x: |x - (m + s code)| <= s / 2.
#include <cuda_runtime.h>

#include "common.cuh"
#include "device_once.h"
#include "kernels.h"

namespace uocr {

__device__ __forceinline__ float bf16_low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_high(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// Values of larger magnitude are refused, so that no difference, step or
// product above overflows.
__device__ __forceinline__ bool kvq_in_range(float x) {
  return fabsf(x) < 1.2676506e30f;  // 2^100; false for NaN
}

// Step and least value of a group from its extremes, packed (s low, m high).
__device__ __forceinline__ uint32_t kvq_params(float lo, float hi, double inv_levels, double levels,
                                               float* s_out, float* m_out) {
  // largest bf16 <= lo: truncation is towards zero, so negatives round up in magnitude
  const uint32_t lb = __float_as_uint(lo);
  const uint32_t mb = (lb & 0x80000000u ? lb + 0xFFFFu : lb) & 0xFFFF0000u;
  const float m = __uint_as_float(mb);
  // d / levels correctly rounded from the rounded reciprocal: one product, its
  // exact remainder and one correction (Markstein, 1990)
  const double d = __dsub_rn(static_cast<double>(hi), static_cast<double>(m));
  const double q = __dmul_rn(d, inv_levels);
  const double t = __fma_rn(__fma_rn(-levels, q, d), inv_levels, q);
  // smallest bf16 >= t (t >= 0): up to float, then up to bf16
  const uint32_t sb = (__float_as_uint(__double2float_ru(t)) + 0xFFFFu) & 0xFFFF0000u;
  *s_out = __uint_as_float(sb);
  *m_out = m;
  return (sb >> 16) | mb;
}

// Code of x: in float, and in double where the float quotient is too near a
// border between two codes (or the step too small) to decide.  The float
// quotient is off by at most 3 roundings of 2^-24, so by 5e-5 at 255.
__device__ __forceinline__ int kvq_code(float x, float m, float s, float inv_s, int levels) {
  const float t = __fmul_rn(__fsub_rn(x, m), inv_s);
  const float r = rintf(t);
  int c = static_cast<int>(r);
  if (!(fabsf(t - r) < 0.4999f) || s < 1e-30f)
    c = s > 0.0f ? __double2int_rn(__ddiv_rn(__dsub_rn(static_cast<double>(x), static_cast<double>(m)),
                                             static_cast<double>(s)))
                 : 0;
  return min(max(c, 0), levels);
}

// One head's row of a key (VALUE false) or value into token t of a tile, by
// one warp, lane = dim of the group: x(d) gives the row.
template <bool VALUE, class Row>
__device__ __forceinline__ void kvq_write_row(unsigned char* tile, const KvqLayout& L, int t, Row x,
                                              unsigned* status) {
  const int lane = threadIdx.x & 31;
  const int levels = (1 << L.bits) - 1;
  const double dl = levels, inv = __ddiv_rn(1.0, dl);
  unsigned char* codes = tile + (VALUE ? L.half : 0);
  for (int grp = 0; grp < L.groups; ++grp) {
    const int d = grp * kKvqGroup + lane;
    const bool in = d < L.dim;
    const float v = in ? x(d) : 0.0f;
    const bool bad = __any_sync(0xffffffffu, in && !kvq_in_range(v));
    float lo = in ? v : INFINITY, hi = in ? v : -INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    float s, m;
    uint32_t word = kvq_params(lo, hi, inv, dl, &s, &m);
    int c = in ? kvq_code(v, m, s, __fdiv_rn(1.0f, s), levels) : 0;
    if (bad) {  // the group reads as NaN
      word = 0x7FC00000u;
      c = 0;
      if (lane == 0) flag(status, DEV_KV_RANGE);
    }
    const int at = VALUE ? kvq_value_byte(t, d, L.bits) : kvq_key_byte(t, d, L.bits);
    if (L.bits == 4) {
      const int up = VALUE ? 8 : 16;  // the dim whose code is the high nibble
      const int high = __shfl_xor_sync(0xffffffffu, c, up);
      if (!(lane & up)) codes[at] = static_cast<unsigned char>(c | (high << 4));
    } else {
      codes[at] = static_cast<unsigned char>(c);
    }
    if (lane == 0) *reinterpret_cast<uint32_t*>(codes + L.codes + kvq_param_byte(t, grp)) = word;
  }
}

__device__ __forceinline__ unsigned char* kvq_tile(unsigned char* data, const KvqLayout& L, int seq,
                                                   int head, long long slot) {
  return data + ((static_cast<long long>(seq) * L.heads + head) * L.tiles + (slot >> 5)) * L.tile;
}

// A prompt's rows: one warp per (token, head).
__global__ void __launch_bounds__(256)
    kvq_prefill_kernel(unsigned char* data, const KvqLayout L, int* state, int seq,
                       const float* __restrict__ k, long long ld_k, const float* __restrict__ v,
                       long long ld_v, int tokens, unsigned* status) {
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    state[2 * seq] = tokens;
    state[2 * seq + 1] = 0;
  }
  const long long rows = static_cast<long long>(tokens) * L.heads;
  for (long long r = blockIdx.x * 8LL + (threadIdx.x >> 5); r < rows; r += gridDim.x * 8LL) {
    const int t = static_cast<int>(r / L.heads), h = static_cast<int>(r % L.heads);
    unsigned char* tile = kvq_tile(data, L, seq, h, t);
    const float* kr = k + t * ld_k + static_cast<long long>(h) * L.dim;
    const float* vr = v + t * ld_v + static_cast<long long>(h) * L.dim;
    kvq_write_row<false>(tile, L, t & 31, [&](int d) { return kr[d]; }, status);
    kvq_write_row<true>(tile, L, t & 31, [&](int d) { return vr[d]; }, status);
  }
}

void launch_kvq_prefill(unsigned char* data, const KvqLayout& L, int* state, int seq, const float* k,
                        long long ld_k, const float* v, long long ld_v, int tokens,
                        unsigned* status, int sms, cudaStream_t st) {
  const long long rows = static_cast<long long>(tokens) * L.heads;
  const long long blocks = (rows + 7) / 8, most = 16LL * sms;
  kvq_prefill_kernel<<<static_cast<int>(blocks < most ? blocks : most), 256, 0, st>>>(
      data, L, state, seq, k, ld_k, v, ld_v, tokens, status);
}

// One token of every sequence: one CTA per sequence, one warp per head and
// turn.  ROPE: rows are the fused projections [q | k | v]; q is rotated into
// q_out and k rotated before it is quantised.
template <bool ROPE>
__global__ void __launch_bounds__(1024)
    kvq_push_kernel(unsigned char* data, const KvqLayout L, int* state, int window,
                    const float* __restrict__ k, long long ld_k, const float* __restrict__ v,
                    long long ld_v, float* q_out, const float2* __restrict__ table, int max_pos,
                    unsigned* status) {
  pdl_launch_dependents();  // launched as a programmatic dependent (launch_dependent):
  pdl_wait_prior_grids();   // nothing is touched before the previous kernel completes
  const int b = blockIdx.x;
  const int prefix = state[2 * b], gen = state[2 * b + 1];
  if (prefix <= 0) {
    if (threadIdx.x == 0) flag(status, DEV_CACHE);
    return;
  }
  const int pos = prefix + gen;
  const long long slot = prefix + gen % window;
  const int half = L.dim >> 1;
  const long long width = static_cast<long long>(L.heads) * L.dim;
  const bool turn = ROPE && pos >= 0 && pos < max_pos;
  if (ROPE && !turn && threadIdx.x == 0) flag(status, DEV_POSITION);
  const float2* cs = ROPE ? table + static_cast<long long>(pos) * half : nullptr;
  // element d of a row, rotated (one rounding per operation, as uocr_kv_rope)
  auto rotated = [&](const float* row, int d) {
    if (!turn) return row[d];
    const int i = d < half ? d : d - half;
    const float2 c = cs[i];
    const float x0 = row[i], x1 = row[i + half];
    return d < half ? __fsub_rn(__fmul_rn(x0, c.x), __fmul_rn(x1, c.y))
                    : __fadd_rn(__fmul_rn(x1, c.x), __fmul_rn(x0, c.y));
  };
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  for (int task = warp; task < 2 * L.heads; task += warps) {
    const int h = task >> 1;
    unsigned char* tile = kvq_tile(data, L, b, h, slot);
    const long long off = static_cast<long long>(h) * L.dim;
    if (task & 1) {
      const float* row = v + b * ld_v + off;
      kvq_write_row<true>(tile, L, slot & 31, [&](int d) { return row[d]; }, status);
    } else {
      const float* row = k + b * ld_k + off;
      kvq_write_row<false>(tile, L, slot & 31,
                           [&](int d) { return ROPE ? rotated(row, d) : row[d]; }, status);
      if (ROPE) {
        const float* q = k - width + b * ld_k + off;
        for (int d = lane; d < L.dim; d += 32) q_out[b * width + off + d] = rotated(q, d);
      }
    }
  }
  __syncthreads();  // every thread has read `gen`
  if (threadIdx.x == 0) state[2 * b + 1] = gen + 1;
}

static int push_threads(const KvqLayout& L) { return 32 * (2 * L.heads < 32 ? 2 * L.heads : 32); }

void launch_kvq_push(unsigned char* data, const KvqLayout& L, int* state, int batch, int window,
                     const float* k, long long ld_k, const float* v, long long ld_v,
                     unsigned* status, cudaStream_t st) {
  launch_dependent(kvq_push_kernel<false>, dim3(batch), dim3(push_threads(L)), 0, st, data, L, state,
                   window, k, ld_k, v, ld_v, nullptr, nullptr, 0, status);
}

void launch_kvq_rope_push(unsigned char* data, const KvqLayout& L, int* state, int batch, int window,
                          const float* qkv, float* q_out, const float2* table, int max_pos,
                          unsigned* status, cudaStream_t st) {
  const long long width = static_cast<long long>(L.heads) * L.dim;
  launch_dependent(kvq_push_kernel<true>, dim3(batch), dim3(push_threads(L)), 0, st, data, L, state,
                   window, qkv + width, 3 * width, qkv + 2 * width, 3 * width, q_out, table, max_pos,
                   status);
}

__device__ __forceinline__ int kvq_tokens(const int* state, int b, int window) {
  const int prefix = state[2 * b], gen = state[2 * b + 1];
  return prefix > 0 ? prefix + (gen < window ? gen : window) : 0;
}

// Slots [first, first + count) of one sequence as token-major rows of floats.
__global__ void __launch_bounds__(256)
    kvq_read_kernel(const unsigned char* __restrict__ data, const KvqLayout L,
                    const int* __restrict__ state, int window, int seq, long long first,
                    long long count, float* k, float* v, unsigned* status) {
  const long long left = kvq_tokens(state, seq, window) - first;
  if (left < count && blockIdx.x == 0 && threadIdx.x == 0) flag(status, DEV_KV_SLOT);
  const long long n = left < count ? left : count;
  const int width = L.heads * L.dim;
  for (long long t = blockIdx.x; t < n; t += gridDim.x) {
    const long long slot = first + t;
    const int tt = static_cast<int>(slot & 31);
    for (int i = threadIdx.x; i < width; i += blockDim.x) {
      const int h = i / L.dim, d = i - h * L.dim;
      const unsigned char* tile = kvq_tile(const_cast<unsigned char*>(data), L, seq, h, slot);
      for (int part = 0; part < 2; ++part) {
        const unsigned char* codes = tile + part * L.half;
        int c = codes[part ? kvq_value_byte(tt, d, L.bits) : kvq_key_byte(tt, d, L.bits)];
        if (L.bits == 4) c = (c >> (4 * (part ? kvq_value_nibble(d) : kvq_key_nibble(d)))) & 15;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + L.codes + kvq_param_byte(tt, d >> 5));
        (part ? v : k)[t * width + i] = __fmaf_rn(bf16_low(w), static_cast<float>(c), bf16_high(w));
      }
    }
  }
}

void launch_kvq_read(const unsigned char* data, const KvqLayout& L, const int* state, int window,
                     int seq, long long first, long long count, float* k, float* v, unsigned* status,
                     int sms, cudaStream_t st) {
  const long long most = 8LL * sms;
  kvq_read_kernel<<<static_cast<int>(count < most ? count : most), 256, 0, st>>>(
      data, L, state, window, seq, first, count, k, v, status);
}

// ---- attention -------------------------------------------------------------------
// One CTA per (head, sequence), four warps that take the tiles in turn, each
// with its own running maximum, sum and weighted values, joined at the end.
constexpr int kKvqWarps = 4;

__global__ void __launch_bounds__(kKvqWarps * 32) kvq_attention_kernel(const KvqAttnArgs a) {
  __shared__ float qs[kKvqMaxDim];
  __shared__ float s_m[kKvqWarps], s_l[kKvqWarps];
  __shared__ float s_o[kKvqWarps][kKvqMaxDim];
  const KvqLayout& L = a.layout;
  const int h = blockIdx.x, b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int T = kvq_tokens(a.state, b, a.window);
  if (T <= 0) {
    if (threadIdx.x == 0) flag(a.status, DEV_CACHE);
    return;
  }
  const long long row = (static_cast<long long>(b) * L.heads + h) * L.dim;
  for (int d = threadIdx.x; d < L.dim; d += blockDim.x) qs[d] = a.q[row + d];
  __syncthreads();
  float m = -INFINITY, l = 0.0f, o[kKvqMaxDim / 32];
  for (int g = 0; g < kKvqMaxDim / 32; ++g) o[g] = 0.0f;
  for (int i = warp; i < (T + 31) / 32; i += kKvqWarps) {
    const unsigned char* kc = kvq_tile(const_cast<unsigned char*>(a.data), L, b, h, 32LL * i);
    const unsigned char* vc = kc + L.half;
    const bool in = 32 * i + lane < T;
    float x = 0.0f;
    for (int g = 0; g < L.groups; ++g) {
      float dot = 0.0f, sum = 0.0f;
      for (int d = 32 * g; d < min(32 * g + 32, L.dim); ++d) {
        int c = kc[kvq_key_byte(lane, d, L.bits)];
        if (L.bits == 4) c = (c >> (4 * kvq_key_nibble(d))) & 15;
        dot = fmaf(qs[d], static_cast<float>(c), dot);
        sum += qs[d];
      }
      const uint32_t w = *reinterpret_cast<const uint32_t*>(kc + L.codes + kvq_param_byte(lane, g));
      x = fmaf(bf16_low(w), dot, fmaf(bf16_high(w), sum, x));
    }
    x = in ? x * a.scale : -INFINITY;
    const float mx = fmaxf(m, warp_max(x));
    const float p = in ? expf(x - mx) : 0.0f, keep = m == -INFINITY ? 0.0f : expf(m - mx);
    m = mx;
    l = l * keep + warp_sum(p);
    for (int g = 0; g < L.groups; ++g) {
      const int d = 32 * g + lane;
      float acc = 0.0f;
      for (int t = 0; t < min(32, T - 32 * i); ++t) {
        const float pt = __shfl_sync(0xffffffffu, p, t);
        int c = vc[kvq_value_byte(t, d, L.bits)];
        if (L.bits == 4) c = (c >> (4 * kvq_value_nibble(d))) & 15;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(vc + L.codes + kvq_param_byte(t, g));
        acc = fmaf(pt, fmaf(bf16_low(w), static_cast<float>(c), bf16_high(w)), acc);
      }
      o[g] = fmaf(o[g], keep, acc);
    }
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  for (int g = 0; g < L.groups; ++g) s_o[warp][32 * g + lane] = o[g];
  __syncthreads();
  float mx = s_m[0];
  bool bad = false;
  for (int w = 0; w < kKvqWarps; ++w) mx = fmaxf(mx, s_m[w]);
  float sum = 0.0f, f[kKvqWarps];
  for (int w = 0; w < kKvqWarps; ++w) {
    f[w] = s_m[w] == -INFINITY && s_l[w] == 0.0f ? 0.0f : expf(s_m[w] - mx);
    sum += f[w] * s_l[w];
  }
  bad = !(sum > 0.0f) || !isfinite(sum) || !isfinite(mx);
  if (bad && threadIdx.x == 0) flag(a.status, DEV_SOFTMAX);
  for (int d = threadIdx.x; d < L.dim; d += blockDim.x) {
    float acc = 0.0f;
    for (int w = 0; w < kKvqWarps; ++w)
      if (f[w] != 0.0f) acc = fmaf(f[w], s_o[w][d], acc);
    a.out[row + d] = bad ? __uint_as_float(0x7FC00000u) : acc / sum;
  }
}

cudaError_t launch_kvq_attention(const KvqAttnArgs& a, int batch, cudaStream_t st) {
  kvq_attention_kernel<<<dim3(a.layout.heads, batch), kKvqWarps * 32, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace uocr
