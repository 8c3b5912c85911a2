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
//
// Every kernel here may be resident while the kernel in front still writes what it
// reads (programmatic dependent launches), so that nothing but a kernel's own
// arguments is read-only for its whole life: loads are plain ones behind the wait,
// never through the non-coherent path (no __ldg, no const __restrict__).
#include <cuda_runtime.h>

#include "common.cuh"
#include "device_once.h"
#include "kernels.h"

namespace uocr {

__device__ __forceinline__ float bf16_low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_high(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

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

// 1 / x within 2^-24 of it: one step of Newton's from an approximation (1 ulp);
// subnormals count as 0.
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return __fmaf_rn(__fmaf_rn(-x, y, 1.0f), y, y);
}

// Largest and least of three and of two; NaN where one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max3_abs(float a, float b, float c) {  // of magnitudes; NaN is none
  float d;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// A group whose extremes hi and -lo are not both below 2^100 in magnitude, or are
// NaN, is refused.
__device__ __forceinline__ bool kvq_refused(float hi, float neg_lo) {
  return !(fmaxf(hi, neg_lo) < 1.2676506e30f) || isnan(hi) || isnan(neg_lo);
}

constexpr float kKvqTinyStep = 1e-30f;  // steps below it (0 among them) go by double

// Codes of four values as the bytes of a word: in float, rounded by adding
// 1.5 2^23 (whose last place is 1).  *near is raised to how far the quotients are from
// their codes.  The float quotient is off by the roundings of the difference and of
// the reciprocal, 2^-23 of it (and a place of the rest, 2^-26), so by 3.1e-5 at 255 and
// 1.9e-6 at 15: from kvq_near on it is too near a border between two codes to decide.
constexpr float kvq_near(int bits) { return bits == 4 ? 0.499998f : 0.499969f; }
__device__ __forceinline__ uint32_t kvq_codes4(const float (&x)[4], float m, float inv_s, float* near) {
  const float2 nm = make_float2(-m, -m), is = make_float2(inv_s, inv_s);
  const float2 magic = make_float2(12582912.0f, 12582912.0f), one = make_float2(-1.0f, -1.0f);
  const float2 d0 = f2_add(make_float2(x[0], x[1]), nm), d1 = f2_add(make_float2(x[2], x[3]), nm);
  const float2 r0 = f2_fma(d0, is, magic), r1 = f2_fma(d1, is, magic);
  const float2 o0 = f2_fma(d0, is, f2_fma(r0, one, magic)), o1 = f2_fma(d1, is, f2_fma(r1, one, magic));
  *near = max3_abs(max3_abs(*near, o0.x, o0.y), o1.x, o1.y);
  return __byte_perm(__byte_perm(__float_as_uint(r0.x), __float_as_uint(r0.y), 0x0040),
                     __byte_perm(__float_as_uint(r1.x), __float_as_uint(r1.y), 0x0040), 0x5410);
}

// The same by the definition, in double (the four divisions in step: a warp that comes
// here holds up its CTA; one by one they cost 2 us more for 32,768 tokens in 8 bits).
__device__ __noinline__ uint32_t kvq_codes4_exactly(float x0, float x1, float x2, float x3, float m,
                                                    float s, int levels) {
  const float x[4] = {x0, x1, x2, x3};
  uint32_t c = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int v = 0;
    if (s > 0.0f)
      v = __double2int_rn(__ddiv_rn(__dsub_rn(static_cast<double>(x[i]), static_cast<double>(m)),
                                    static_cast<double>(s)));
    c |= static_cast<uint32_t>(min(max(v, 0), levels)) << (8 * i);
  }
  return c;
}

// Four values of a row from dim d (a multiple of 4); zeros past the row's end.
template <bool VEC>
__device__ __forceinline__ void kvq_load4(const float* row, int d, int dim, float (&x)[4]) {
  if (VEC) {
    const float4 v = d < dim ? *reinterpret_cast<const float4*>(row + d)
                             : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    x[0] = v.x;
    x[1] = v.y;
    x[2] = v.z;
    x[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = d + i < dim ? row[d + i] : 0.0f;
  }
}

__device__ __forceinline__ unsigned char* kvq_tile(unsigned char* data, const KvqLayout& L, int seq,
                                                   int head, long long slot) {
  return data + ((static_cast<long long>(seq) * L.heads + head) * L.tiles + (slot >> 5)) * L.tile;
}

__global__ void kvq_reset_kernel(int* state, int seq) {
  pdl_launch_dependents();
  pdl_wait_prior_grids();
  state[2 * seq] = state[2 * seq + 1] = 0;
}

void launch_kvq_reset(int* state, int seq, cudaStream_t st) {
  launch_dependent(kvq_reset_kernel, dim3(1), dim3(1), 0, st, state, seq);
}

// ---- a prompt's rows ------------------------------------------------------------
// One CTA per (tile, head), one warp per four tokens: of the keys every eighth, whose
// codes are one 16-byte unit of a plane, of the values neighbours, so that the bytes of
// a value word (four tokens of one dim) meet in one lane.  Eight lanes share a group,
// four dims each; four groups at a time.  The extremes of four tokens are eight values
// over eight lanes: halving what a lane keeps at every exchange takes 7 shuffles instead
// of 24 and leaves the extremes of token u in the lanes u and u + 4 of the eight, which
// then find its parameters once.
// Bound by the bytes of the rows and, nearly as much, by issue (70 % of the slots) and
// the latency of a CTA's load - compute - copy chain: 32,768 tokens of 10 heads of 128
// take 69.0 us in 4 bits (388 MB: 5.6 TB/s) and 74.3 us in 8 bits (430 MB: 5.8 TB/s),
// the reset before it counted in.  Six CTAs per SM leave 40 registers and cost 120 to
// 128 bytes of spills a thread; five CTAs (48 registers, 56 to 104 bytes) take 70.7 and
// 76.2 us.  An earlier form of 87 us (8 bits) took 104 in
// persistent CTAs whose rows arrive by asynchronous copies while they work on the last
// ones.
// VEC: rows that four floats at a time can be read from, so that a lane's four dims
// are the row's or not as one.
template <int BITS, bool VEC>
__global__ void __launch_bounds__(256, 6)
    kvq_prefill_kernel(unsigned char* data, const KvqLayout L, int* state, int seq,
                       const float* k, long long ld_k, const float* v, long long ld_v, int tokens,
                       unsigned* status) {
  extern __shared__ __align__(128) unsigned char kvq_stage[];
  pdl_launch_dependents();  // launched as a programmatic dependent (launch_dependent):
  pdl_wait_prior_grids();   // nothing is touched before the previous kernel completes
  constexpr int levels = (1 << BITS) - 1;
  const int h = blockIdx.x % L.heads, tile = blockIdx.x / L.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l8 = lane & 7;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    state[2 * seq] = tokens;
    state[2 * seq + 1] = 0;
  }
  const int half = warp >> 2, j = warp & 3;
  const bool h4 = l8 & 4, h2 = l8 & 2, h1 = l8 & 1;
  for (int q = 0; q < (L.groups + 3) / 4; ++q) {
    const int grp = q * 4 + (lane >> 3), d0 = grp * 32 + l8 * 4;
    const bool real = grp < L.groups;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      // this warp's tokens: for keys each eighth, so that they are one 16-byte unit, for
      // values neighbours, the bytes of a word
      const int first = tile * 32 + (part ? warp * 4 : warp), step = part ? 1 : 8;
      const long long ld = part ? ld_v : ld_k;
      const float* row = (part ? v : k) + first * ld + static_cast<long long>(h) * L.dim;
      float x[4][4];
#pragma unroll
      for (int u = 0; u < 4; ++u, row += step * ld) {
        if (first + step * u < tokens) {
          kvq_load4<VEC>(row, d0, L.dim, x[u]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[u][i] = 0.0f;
        }
      }
      // the largest x and the largest -x of each token, over this lane's dims
      float a[4], b[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        a[u] = b[u] = -INFINITY;
        if (VEC) {
          if (d0 < L.dim) {
            a[u] = max_nan(max3_nan(x[u][0], x[u][1], x[u][2]), x[u][3]);
            b[u] = max_nan(-min3_nan(x[u][0], x[u][1], x[u][2]), -x[u][3]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (d0 + i < L.dim) {
              a[u] = max_nan(a[u], x[u][i]);
              b[u] = max_nan(b[u], -x[u][i]);
            }
        }
      }
      float e[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        e[u] = max_nan(h4 ? b[u] : a[u], __shfl_xor_sync(0xffffffffu, h4 ? a[u] : b[u], 4));
      const float e0 = max_nan(h2 ? e[2] : e[0], __shfl_xor_sync(0xffffffffu, h2 ? e[0] : e[2], 2));
      const float e1 = max_nan(h2 ? e[3] : e[1], __shfl_xor_sync(0xffffffffu, h2 ? e[1] : e[3], 2));
      const float mine = max_nan(h1 ? e1 : e0, __shfl_xor_sync(0xffffffffu, h1 ? e0 : e1, 1));
      const float other = __shfl_xor_sync(0xffffffffu, mine, 4);
      const bool lost = real && kvq_refused(mine, other);  // of token l8 & 3: it reads as NaN
      float s, m;
      uint32_t word = kvq_params(-(h4 ? mine : other), h4 ? other : mine, 1.0 / levels, levels, &s, &m);
      const float inv_s = rcp_fast(s);
      if (lost) word = 0x7FC00000u;
      unsigned char* codes = kvq_stage + part * L.half;
      if (real && l8 < 4)
        *reinterpret_cast<uint32_t*>(codes + L.codes + kvq_param_byte(part ? warp * 4 + l8 : warp + 8 * l8, grp)) = word;
      uint32_t c[4];
      float near = 0.0f;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        c[u] = kvq_codes4(x[u], __shfl_sync(0xffffffffu, m, (lane & 24) + u),
                          __shfl_sync(0xffffffffu, inv_s, (lane & 24) + u), &near);
      // (rare: 3 warps in 100 at 8 bits)
      const bool some = d0 < L.dim;
      if (__any_sync(0xffffffffu, (some && near >= kvq_near(BITS)) || (real && s < kKvqTinyStep) || lost)) {
        if (lost) flag(status, DEV_KV_RANGE);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int from = (lane & 24) + u;
          const float mu = __shfl_sync(0xffffffffu, m, from), su = __shfl_sync(0xffffffffu, s, from);
          near = 0.0f;
          c[u] = kvq_codes4(x[u], mu, __shfl_sync(0xffffffffu, inv_s, from), &near);
          if (some && (near >= kvq_near(BITS) || su < kKvqTinyStep))
            c[u] = kvq_codes4_exactly(x[u][0], x[u][1], x[u][2], x[u][3], mu, su, levels);
          if (__shfl_sync(0xffffffffu, lost, from)) c[u] = 0;
        }
      }
      if (d0 + 3 >= L.dim) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (d0 + i >= L.dim) c[u] &= ~(0xFFu << (8 * i));
      }
      if (part == 0) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (BITS == 4) c[u] |= __shfl_xor_sync(0xffffffffu, c[u], 4) << 4;
          c[u] ^= kvq_flip(BITS);
        }
        if (real && (BITS == 8 || !h4))
          *reinterpret_cast<uint4*>(codes + kvq_key_byte(warp, d0, BITS)) = make_uint4(c[0], c[1], c[2], c[3]);
      } else {
        // bytes: token u of dim i; as words: dim i of the four tokens
        const uint32_t lo = __byte_perm(c[0], c[1], 0x5140), hi = __byte_perm(c[0], c[1], 0x7362);
        const uint32_t lo2 = __byte_perm(c[2], c[3], 0x5140), hi2 = __byte_perm(c[2], c[3], 0x7362);
        uint32_t w[4] = {__byte_perm(lo, lo2, 0x5410), __byte_perm(lo, lo2, 0x7632),
                         __byte_perm(hi, hi2, 0x5410), __byte_perm(hi, hi2, 0x7632)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (BITS == 4) w[i] |= __shfl_xor_sync(0xffffffffu, w[i], 2) << 4;
          w[i] ^= kvq_flip(BITS);
        }
        // (word i lies 64 i bytes from the first: half of the lanes of a bank take them in
        // another order, 4 us less for 32,768 tokens in 8 bits)
        const bool turn = lane & 8;
        unsigned char* at = codes + kvq_value_byte(half * 16 + j * 4, d0, BITS);
        if (real && (BITS == 8 || !h2)) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint32_t*>(at + (turn ? (i ^ 1) * 64 : i * 64)) = turn ? w[i ^ 1] : w[i];
        }
      }
    }
  }
  // the tile leaves as one bulk copy (8 us less than vector stores of all threads)
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncthreads();
  // (slots past the prompt's end in its last tile get zeros: nothing is in them)
  if (threadIdx.x == 0) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                     kvq_tile(data, L, seq, h, tile * 32LL)),
                 "r"(smem_addr(kvq_stage)), "r"(static_cast<uint32_t>(L.tile))
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
}

// Rows that four floats at a time can be read from (or written to).
static bool kvq_vec(const KvqLayout& L, const void* k, long long ld_k, const void* v, long long ld_v) {
  return L.dim % 4 == 0 && ld_k % 4 == 0 && ld_v % 4 == 0 && reinterpret_cast<uintptr_t>(k) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(v) % 16 == 0;
}

void launch_kvq_prefill(unsigned char* data, const KvqLayout& L, int* state, int seq, const float* k,
                        long long ld_k, const float* v, long long ld_v, int tokens,
                        unsigned* status, cudaStream_t st) {
  const unsigned blocks = static_cast<unsigned>((tokens + 31) / 32) * L.heads;
  const bool vec = kvq_vec(L, k, ld_k, v, ld_v);
  auto kernel = L.bits == 4 ? vec ? kvq_prefill_kernel<4, true> : kvq_prefill_kernel<4, false>
                : vec       ? kvq_prefill_kernel<8, true>
                            : kvq_prefill_kernel<8, false>;
  launch_dependent(kernel, dim3(blocks), dim3(256), static_cast<size_t>(L.tile), st, data, L, state, seq, k,
                   ld_k, v, ld_v, tokens, status);
}

// ---- one token of every sequence ----------------------------------------------------
// One CTA per sequence, one warp per head and key or value; lanes as above, the token's
// bytes straight into the tile.  ROPE: the rows are the fused projections [q | k | v];
// q is rotated into q_out and k rotated before it is quantised.  Bound by the latency
// of a launch and two dependent loads: 2.4 us in a chain of launches, for 1 sequence as
// for 64.
constexpr int kKvqPushWarps = 20;

template <int BITS, bool ROPE>
__global__ void __launch_bounds__(kKvqPushWarps * 32)
    kvq_push_kernel(unsigned char* data, const KvqLayout L, int* state, int window,
                    const float* k, long long ld_k, const float* v, long long ld_v, float* q_out,
                    const float2* table, int max_pos, unsigned* status) {
  constexpr int levels = (1 << BITS) - 1;
  pdl_launch_dependents();  // launched as a programmatic dependent (launch_dependent):
  pdl_wait_prior_grids();   // nothing is touched before the previous kernel completes
  const int b = blockIdx.x;
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31, l8 = lane & 7;
  const int half = L.dim >> 1;
  const long long width = static_cast<long long>(L.heads) * L.dim;
  // A lane's four dims of task's row from dim d0, and what they are rotated with.
  float x[4], y[4];
  auto load = [&](int task, int d0) {
    const bool value = task & 1;
    const float* row = (value ? v + b * ld_v : k + b * ld_k) + static_cast<long long>(task >> 1) * L.dim;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = d0 + i;
      x[i] = d < L.dim ? row[d] : 0.0f;
      if (ROPE && !value) y[i] = d < L.dim ? row[d < half ? d + half : d - half] : 0.0f;
    }
  };
  // (the first rows and the state arrive together)
  if (warp < 2 * L.heads) load(warp, (lane >> 3) * 32 + l8 * 4);
  const int prefix = state[2 * b], gen = state[2 * b + 1];
  if (prefix <= 0) {
    if (threadIdx.x == 0) flag(status, DEV_CACHE);
    return;
  }
  const int pos = prefix + gen;
  const long long slot = prefix + gen % window;
  const int t = static_cast<int>(slot & 31);
  const bool turn = ROPE && pos >= 0 && pos < max_pos;
  if (ROPE && !turn && threadIdx.x == 0) flag(status, DEV_POSITION);
  const float2* cs = ROPE ? table + static_cast<long long>(pos) * half : nullptr;
  // element d of a row, x0, rotated with x1, half a row from it (one rounding per
  // operation, as uocr_kv_rope)
  auto rotated = [&](float x0, float x1, int d) {
    if (!turn) return x0;
    const float2 c = cs[d < half ? d : d - half];
    return d < half ? __fsub_rn(__fmul_rn(x0, c.x), __fmul_rn(x1, c.y))
                    : __fadd_rn(__fmul_rn(x0, c.x), __fmul_rn(x1, c.y));
  };
  for (int task = warp; task < 2 * L.heads; task += warps) {
    const int h = task >> 1;
    const bool value = task & 1;
    const long long off = static_cast<long long>(h) * L.dim;
    unsigned char* codes = kvq_tile(data, L, b, h, slot) + (value ? L.half : 0);
    for (int q = 0; q < (L.groups + 3) / 4; ++q) {
      const int grp = q * 4 + (lane >> 3), d0 = grp * 32 + l8 * 4;
      const bool real = grp < L.groups;
      if (task != warp || q) load(task, d0);
      float hi = -INFINITY, neg_lo = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = d0 + i;
        if (d < L.dim) {
          if (ROPE && !value) x[i] = rotated(x[i], y[i], d);
          hi = max_nan(hi, x[i]);
          neg_lo = max_nan(neg_lo, -x[i]);
        }
      }
#pragma unroll
      for (int o = 1; o <= 4; o <<= 1) {
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        neg_lo = max_nan(neg_lo, __shfl_xor_sync(0xffffffffu, neg_lo, o));
      }
      float s, m, near = 0.0f;
      uint32_t word = kvq_params(-neg_lo, hi, 1.0 / levels, levels, &s, &m);
      uint32_t c = kvq_codes4(x, m, rcp_fast(s), &near);
      if (near >= kvq_near(BITS) || s < kKvqTinyStep) c = kvq_codes4_exactly(x[0], x[1], x[2], x[3], m, s, levels);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (d0 + i >= L.dim) c &= ~(0xFFu << (8 * i));
      if (real && kvq_refused(hi, neg_lo)) {  // reads as NaN
        word = 0x7FC00000u;
        c = 0;
        flag(status, DEV_KV_RANGE);
      }
      if (real && l8 == 0) *reinterpret_cast<uint32_t*>(codes + L.codes + kvq_param_byte(t, grp)) = word;
      const uint32_t up = __shfl_xor_sync(0xffffffffu, c, value ? 2 : 4);
      if (BITS == 4) c |= up << 4;
      c ^= kvq_flip(BITS);
      if (!real || (BITS == 4 && (l8 & (value ? 2 : 4)))) continue;
      if (!value) {
        *reinterpret_cast<uint32_t*>(codes + kvq_key_byte(t, d0, BITS)) = c;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          codes[kvq_value_byte(t, d0 + i, BITS)] = static_cast<unsigned char>(c >> (8 * i));
      }
    }
    if (ROPE && !value) {
      const float* q = k - width + b * ld_k + off;
      for (int d = lane; d < L.dim; d += 32)
        q_out[b * width + off + d] = rotated(q[d], q[d < half ? d + half : d - half], d);
    }
  }
  __syncthreads();  // every thread has read `gen`
  if (threadIdx.x == 0) state[2 * b + 1] = gen + 1;
}

static int push_threads(const KvqLayout& L) {
  return 32 * (2 * L.heads < kKvqPushWarps ? 2 * L.heads : kKvqPushWarps);
}

void launch_kvq_push(unsigned char* data, const KvqLayout& L, int* state, int batch, int window,
                     const float* k, long long ld_k, const float* v, long long ld_v,
                     unsigned* status, cudaStream_t st) {
  launch_dependent(L.bits == 4 ? kvq_push_kernel<4, false> : kvq_push_kernel<8, false>, dim3(batch),
                   dim3(push_threads(L)), 0, st, data, L, state, window, k, ld_k, v, ld_v, nullptr,
                   nullptr, 0, status);
}

void launch_kvq_rope_push(unsigned char* data, const KvqLayout& L, int* state, int batch, int window,
                          const float* qkv, float* q_out, const float2* table, int max_pos,
                          unsigned* status, cudaStream_t st) {
  const long long width = static_cast<long long>(L.heads) * L.dim;
  launch_dependent(L.bits == 4 ? kvq_push_kernel<4, true> : kvq_push_kernel<8, true>, dim3(batch),
                   dim3(push_threads(L)), 0, st, data, L, state, window, qkv + width, 3 * width,
                   qkv + 2 * width, 3 * width, q_out, table, max_pos, status);
}

__device__ __forceinline__ int kvq_tokens(const int* state, int b, int window) {
  const int prefix = state[2 * b], gen = state[2 * b + 1];
  return prefix > 0 ? prefix + (gen < window ? gen : window) : 0;
}

// ---- reading back -----------------------------------------------------------------
// Slots [first, first + count) of one sequence as token-major rows of floats: one CTA
// per (tile, head), the tile staged in shared memory, lanes as in the prompt's kernel.
// Bound by the rows written: 32,768 tokens of 10 heads of 128 take 62 us from 4 bits
// and 69 us from 8 (6.2 and 6.3 TB/s).  With six CTAs per SM; five took 71 us from 8
// bits and eight 73.
template <int BITS, bool VEC>
__global__ void __launch_bounds__(256, 6)
    kvq_read_kernel(const unsigned char* data, const KvqLayout L, const int* state, int window, int seq,
                    long long first, long long count, float* k, float* v, unsigned* status) {
  extern __shared__ __align__(128) unsigned char kvq_stage[];
  pdl_launch_dependents();  // launched as a programmatic dependent (launch_dependent):
  pdl_wait_prior_grids();   // nothing is touched before the previous kernel completes
  const int h = blockIdx.x % L.heads;
  const long long tile = (first >> 5) + blockIdx.x / L.heads;
  const uint4* in = reinterpret_cast<const uint4*>(
      kvq_tile(const_cast<unsigned char*>(data), L, seq, h, tile * 32));
  // (three loads in flight per thread: an 8-bit tile of 128 dims in one round)
  for (int i = threadIdx.x; i < L.tile / 16; i += 3 * 256) {
    uint4 w[3];
#pragma unroll
    for (int u = 0; u < 3; ++u)
      if (i + u * 256 < L.tile / 16) w[u] = in[i + u * 256];
#pragma unroll
    for (int u = 0; u < 3; ++u)
      if (i + u * 256 < L.tile / 16) reinterpret_cast<uint4*>(kvq_stage)[i + u * 256] = w[u];
  }
  const long long held = kvq_tokens(state, seq, window);
  const long long end = first + count < held ? first + count : held;
  if (held < first + count && blockIdx.x == 0 && threadIdx.x == 0) flag(status, DEV_KV_SLOT);
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l8 = lane & 7;
  const long long t0 = tile * 32 + warp * 4, width = static_cast<long long>(L.heads) * L.dim;
  for (int q = 0; q < (L.groups + 3) / 4; ++q) {
    const int grp = q * 4 + (lane >> 3), d0 = grp * 32 + l8 * 4;
    if (grp >= L.groups || d0 >= L.dim) continue;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const unsigned char* codes = kvq_stage + part * L.half;
      uint32_t c[4];  // bytes: keys: dims of token u; values: tokens of dim u
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        c[u] = *reinterpret_cast<const uint32_t*>(
            codes + (part ? kvq_value_byte(warp * 4, d0 + u, BITS) : kvq_key_byte(warp * 4 + u, d0, BITS)));
        c[u] ^= kvq_flip(BITS);
        if (BITS == 4) c[u] = (l8 & (part ? 2 : 4) ? c[u] >> 4 : c[u]) & 0x0F0F0F0Fu;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + L.codes + kvq_param_byte(warp * 4 + u, grp));
        const float s = bf16_low(w), m = bf16_high(w);
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = __fmaf_rn(s, static_cast<float>(((part ? c[i] : c[u]) >> (8 * (part ? u : i))) & 0xFFu), m);
        if (t0 + u < first || t0 + u >= end) continue;
        float* row = (part ? v : k) + (t0 + u - first) * width + static_cast<long long>(h) * L.dim + d0;
        if (VEC) {
          *reinterpret_cast<float4*>(row) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (d0 + i < L.dim) row[i] = x[i];
        }
      }
    }
  }
}

void launch_kvq_read(const unsigned char* data, const KvqLayout& L, const int* state, int window,
                     int seq, long long first, long long count, float* k, float* v, unsigned* status,
                     cudaStream_t st) {
  const long long tiles = ((first + count - 1) >> 5) - (first >> 5) + 1;
  const unsigned blocks = static_cast<unsigned>(tiles * L.heads);
  const bool vec = kvq_vec(L, k, 0, v, 0);
  auto kernel = L.bits == 4 ? vec ? kvq_read_kernel<4, true> : kvq_read_kernel<4, false>
                : vec       ? kvq_read_kernel<8, true>
                            : kvq_read_kernel<8, false>;
  launch_dependent(kernel, dim3(blocks), dim3(256), static_cast<size_t>(L.tile), st, data, L, state, window,
                   seq, first, count, k, v, status);
}

// ---- attention -------------------------------------------------------------------
// One query per (head, sequence) over the tiles of its cache.  The codes go to
// the matrix unit nearly as they lie (s8, m16n8k32: c - C with C the middle of the
// codes, 16 (c - 8) for 4 bits), the query and the softmax weights as fixed-point
// numbers cut into bytes, one byte per column of the 8-wide operand, so that every
// product is exact and nothing is dequantised.  With z = m + C s:
//
//   scores:  rows = 16 tokens, k = the 32 dims of a group, columns = the four
//            signed bytes of q 2^a (|q 2^a| < 2^30, a by the group's largest |q|);
//            q . (c - C) = sum_b 256^b D_b, then s (q . (c - C)) + z sum(q), summed
//            from minus the running maximum: a score that counts ends near zero and
//            costs no rounding of its own size;
//   values:  rows = 16 dims, k = the tile's 32 tokens, columns = the four bytes
//            of p_t s_t 2^a (< 2^31, a by the largest p_t s_t of the group so far);
//            o += 2^-a sum_b 256^b D_b, and p_t z_t is summed apart.
//
// Around the middle the sums stay near the size of what they stand for (from 0 up
// they cancel against the least values, which cost a factor of two in accuracy).
// Two neighbouring groups share an accumulator: a group's operand has its bytes
// in its four columns and zeros in the other group's four.  The fixed points keep
// 2^-31 of the group's largest |q| and 2^-31 to 2^-30 of its largest p_t s_t, so
// that what they lose is below a float's rounding of the group's largest term; a
// term that is 2^-7 of that one and less would have kept more in a float of its own.
//
// A tile is one bulk copy.  Every warp has a ring of its own, takes a run of
// neighbouring tiles, and keeps its own maximum, sum and weighted values, so the
// loop has no barrier but the ring's.  The warps' parts are joined in shared
// memory, the CTAs' of a cluster through distributed shared memory, the clusters'
// of a head (where the heads are few) by the one that ends last.
//
// Bound by the cache's bytes where there are many: 64 sequences of 2,176 tokens, 10
// heads of 128, take 39.0 us in 4 bits (222.8 MB: 5.7 TB/s, 4 us of it the start and
// the end of a launch) and 61.6 us in 8 bits (401 MB: 6.5 TB/s), 128 sequences of
// 2,048 tokens 65.0 us in 4 bits (6.5 TB/s); one of 1,645 tokens takes 5.5 us, one of
// 32,768 tokens 15.2 us (7 us without its bytes) and 22.4 us in 8 bits.  The same from
// dequantised values would need some 3 instructions an element, a scheduler's whole
// rate at this bandwidth; here it is about 1.7 an element (ncu: 53 % of the issue slots).
// Not by the tokens of a sequence: the work is split by the cache's capacity and heads,
// so that one sequence of 32,640 tokens among 63 of 500 takes 170 us in 4 bits (64 of
// 1,002, as many tokens, 21.5), and 500 tokens 4.4 us in a cache of 2,048 but 8.2 us in
// one of 32,640.
// Scores are in powers of two.  They may pass the running maximum by this much.
constexpr float kKvqSlack = 2.0f;
// A tile whose scores lie further than this from the maximum that they were summed
// against is summed again, unless a float at that maximum is too coarse for it.
constexpr float kKvqFar = 8.0f, kKvqVast = 1048576.0f;
// Ring slots per warp.  Two tiles in flight for each of 17 warps per SM hide the
// memory better than more for fewer warps (64 x 2,176 tokens, 4 bits, as measured when
// two took 39.4 us: three 46.2, four 52.9).
constexpr int kKvqSlots = 2;
constexpr int kKvqCluster = 8;  // most CTAs of a cluster (portable)

__host__ __device__ constexpr int kvq_tile_bytes(int groups, int bits) {
  return 2 * groups * (512 * (bits / 4) + 128);
}

// Tiles per turn of a warp and per ring slot: two of the smallest tiles (larger ones
// gain nothing by it: 39.9 against 39.2 us for the sizes above).
__host__ __device__ constexpr int kvq_per(int groups, int bits) {
  return kvq_tile_bytes(groups, bits) <= 1280 ? 2 : 1;
}
// Warps of a CTA, by the bytes of its ring: with 128 dims some 45 KB of shared memory (4
// bits) and 39 (8), so that five CTAs share an SM and 740 of them, more than the 640
// heads of a batch of 64, run at once (8 bits, 9 KB tiles: two warps 62.4 us, four
// 71.8).  Other dims were not swept: 24 to 29 KB at 96 (8 bits) and 160.
__host__ __device__ constexpr int kvq_warps(int groups, int bits) {
  const int turn = kvq_tile_bytes(groups, bits) * kvq_per(groups, bits);
  return turn <= 5120 ? 4 : turn <= 10240 ? 2 : 1;
}

template <int G, int BITS>
struct KvqShared {
  static constexpr int W = kvq_warps(G, BITS), N = kvq_per(G, BITS);
  alignas(128) unsigned char ring[W][kKvqSlots][N * kvq_tile_bytes(G, BITS)];
  alignas(16) uint32_t weights[W][N][G][32];
  uint64_t full[W][kKvqSlots];
  float o[W][G * 32];  // weighted values per warp; the CTA's in [0]
  float m[W], l[W];
  float cta_m, cta_l;
  int turn;
};

// s8 rows times signed (SIGNED) or unsigned columns, 32-bit sums.
template <bool SIGNED>
__device__ __forceinline__ void mma_s8_m16n8k32(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                                uint32_t a3, uint32_t b0, uint32_t b1) {
  if (SIGNED)
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 times the signed nibbles of a word, as signed bytes.
__device__ __forceinline__ uint32_t nibbles_low(uint32_t w) { return (w << 4) & 0xF0F0F0F0u; }
__device__ __forceinline__ uint32_t nibbles_high(uint32_t w) { return w & 0xF0F0F0F0u; }

__device__ __forceinline__ float exp2_fast(float x) {  // 2 ulp; exact 1 at 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Byte `byte` of four words as one word.
__device__ __forceinline__ uint32_t gather_bytes(uint32_t x, uint32_t y, uint32_t z, uint32_t w,
                                                 uint32_t byte) {
  const uint32_t sel = byte | ((byte + 4) << 4);
  return __byte_perm(__byte_perm(x, y, sel), __byte_perm(z, w, sel), 0x5410);
}

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float cluster_load(const float* p, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// Factor that a part with maximum m and sum l takes in a whole with maximum M;
// a part without tokens (m = -inf, l = 0) takes none.
__device__ __forceinline__ float part_factor(float m, float l, float M) {
  return m == -INFINITY && l == 0.0f ? 0.0f : exp2_fast(m - M);
}

template <int G, int BITS>
__global__ void __launch_bounds__(kvq_warps(G, BITS) * 32) kvq_attention_kernel(const KvqAttnArgs a) {
  using Shared = KvqShared<G, BITS>;
  constexpr int P = (G + 1) / 2;  // accumulators: pairs of groups
  constexpr int N = Shared::N, W = Shared::W;
  constexpr int kTileBytes = kvq_tile_bytes(G, BITS);
  constexpr int kCodes = G * 512 * (BITS / 4);
  constexpr float kMiddle = 1 << (BITS - 1);
  constexpr int kShift = BITS == 4 ? 4 : 0;  // the operand is 2^kShift (c - kMiddle)
  extern __shared__ __align__(128) unsigned char kvq_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(kvq_raw);
  // a head: `parts` clusters of `splits` CTAs
  const int splits = a.splits, share = blockIdx.x % (splits * a.parts), rank = share % splits;
  const int h = blockIdx.x / (splits * a.parts), b = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  const int workers = splits * a.parts * W, me = share * W + warp;
  const unsigned char* head =
      a.data + (static_cast<long long>(b) * a.layout.heads + h) * a.layout.tiles * kTileBytes;
  auto begin = [&](int tiles, int w) {
    return static_cast<int>(static_cast<long long>(tiles) * w / workers);
  };
  pdl_wait_prior_grids();  // launched as a programmatic dependent (launch_dependent)
  const int T = kvq_tokens(a.state, b, a.window);
  if (T <= 0) {  // the same for every CTA of the cluster
    if (threadIdx.x == 0 && share == 0) flag(a.status, DEV_CACHE);
    return;
  }
  const int tiles = (T + 31) >> 5, first = begin(tiles, me), last = begin(tiles, me + 1);
  const int end = min(T, last * 32);  // this warp's tokens end here
  // tiles it, it + 1 of this warp into ring slot `slot`
  auto fetch = [&](int it, int slot) {
    const uint32_t bytes = (last - it < N ? last - it : N) * kTileBytes;
    mbar_arrive_expect_tx(&sh.full[warp][slot], bytes);
    bulk_g2s(sh.ring[warp][slot], head + static_cast<long long>(it) * kTileBytes, bytes,
             &sh.full[warp][slot]);
  };
  if (lane == 0) {
    for (int i = 0; i < kKvqSlots; ++i) mbar_init(&sh.full[warp][i], 1 + a.wait.extra);
    fence_mbar_init();
    for (int i = 0; i < kKvqSlots && first + i * N < last; ++i) fetch(first + i * N, i);
  }
  __syncwarp();

  // ---- the query's bytes: lane (n, j) of the 8-wide operand holds byte n & 3 of
  // dims 4j .. 4j+3 and 16 + 4j .. of the groups 2a + n / 4, zero of the others
  const int col_group = lane >> 4, col_byte = (lane >> 2) & 3;
  const int acc_group = j >> 1;   // group (of a pair) of this lane's accumulator columns
  const long long row = (static_cast<long long>(b) * a.layout.heads + h) * a.layout.dim;
  uint32_t qb[G][2];
  float qscale[P], qsum[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int grp = 2 * p + col_group;
    float v[8], big = 0.0f;
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = grp * 32 + (i >> 2) * 16 + 4 * j + (i & 3);
      const float qd = d < a.layout.dim ? a.q[row + d] : 0.0f;
      v[i] = fmaf(qd, a.scale_rest, qd * a.scale);  // q log2(e) / sqrt(dim)
      big = fmaxf(big, fabsf(v[i]));
      sum += v[i];
    }
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    // big < 2^(e - 126); a group of magnitudes below 2^-86 loses precision, by
    // scores that are nothing
    const int e = max(static_cast<int>(__float_as_uint(big) >> 23), 40);
    const float up = __uint_as_float(static_cast<uint32_t>(283 - min(e, 254)) << 23);
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)  // signed bytes: byte b of q + 0x808080, flipped, but the top one
      u[i] = (static_cast<uint32_t>(__float2int_rn(v[i] * up)) + 0x00808080u) ^ 0x00808080u;
    const uint32_t lo = gather_bytes(u[0], u[1], u[2], u[3], col_byte);
    const uint32_t hi = gather_bytes(u[4], u[5], u[6], u[7], col_byte);
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (2 * p + c < G) {
        qb[2 * p + c][0] = col_group == c ? lo : 0;
        qb[2 * p + c][1] = col_group == c ? hi : 0;
      }
    // for the accumulators: 2^-a (times 256^2 where the lane holds the upper two
    // bytes) and the sum, its rounding in the other lane: where an outlying dim takes
    // z far from zero, z sum(q) cancels against the upper bytes.  NaN and infinities
    // of q reach the scores by the sum
    const int ea = __shfl_sync(0xffffffffu, e, acc_group * 16);
    const double sa = __shfl_sync(0xffffffffu, sum, acc_group * 16);
    const float most = static_cast<float>(sa);
    const bool real = 2 * p + acc_group < G;
    qscale[p] = real ? __uint_as_float(static_cast<uint32_t>(min(ea, 254) - 29 - kShift + (j & 1) * 16) << 23) : 0.0f;
    qsum[p] = !real ? 0.0f : j & 1 ? most : static_cast<float>(sa - most);
  }

  float m = 0.0f, l = 0.0f, middle[G], o[P][2][2];
  float start = 0.0f;  // of this lane's sums of scores: -m over the lanes of a row
  // per group: the largest weight times step when the fixed point was last set, and
  // what weights are scaled by and their sums scaled back
  float seen[G], wup[G], wdown[P];
#pragma unroll
  for (int i = 0; i < G; ++i) {
    middle[i] = 0.0f;
    seen[i] = 0.0f;
    wup[i] = 0.0f;
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
    wdown[p] = 0.0f;
    o[p][0][0] = o[p][0][1] = o[p][1][0] = o[p][1][1] = 0.0f;
  }

  const int t = g + 8 * j;  // the token of a tile that this lane weighs
  bool again = false;  // this turn's scores are summed a second time
  // no score but -inf so far: m is none of them.  A score of -inf (below the least
  // float) weighs nothing, in this warp or another; a head with no other has no sum
  bool fresh = true;
  for (int it = first, slot = 0, phase = 0; it < last;) {
    if (!__all_sync(0xffffffffu, mbar_wait_try(&sh.full[warp][slot], phase, a.status, a.wait.cycles))) {
      // (a safety net: flagged, the head is NaN) copies in flight land before the CTA ends
      for (int i = 1; i < kKvqSlots && it + i * N < last; ++i) {
        if (++slot == kKvqSlots) {
          slot = 0;
          phase ^= 1;
        }
        mbar_wait_try(&sh.full[warp][slot], phase, a.status, a.wait.cycles);
      }
      l = __uint_as_float(0x7FC00000u);
      break;
    }
    const unsigned char* tile = sh.ring[warp][slot];
    // ---- scores (of a tile past the warp's last: of whatever the slot holds, masked below)
    float score[N];  // against m
    uint32_t par[N][G];
    bool in[N] = {};
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const unsigned char* kt = tile + u * kTileBytes;
      int d[2][P][4];
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[0][p][i] = d[1][p][i] = 0;
#pragma unroll
      for (int grp = 0; grp < G; ++grp) {
        uint4 lo, hi;
        if (BITS == 4) {
          const uint4 w = *reinterpret_cast<const uint4*>(kt + grp * 512 + lane * 16);
          lo = make_uint4(nibbles_low(w.x), nibbles_low(w.y), nibbles_low(w.z), nibbles_low(w.w));
          hi = make_uint4(nibbles_high(w.x), nibbles_high(w.y), nibbles_high(w.z), nibbles_high(w.w));
        } else {
          lo = *reinterpret_cast<const uint4*>(kt + grp * 1024 + lane * 16);
          hi = *reinterpret_cast<const uint4*>(kt + grp * 1024 + 512 + lane * 16);
        }
        mma_s8_m16n8k32<true>(d[0][grp >> 1], lo.x, lo.y, hi.x, hi.y, qb[grp][0], qb[grp][1]);
        mma_s8_m16n8k32<true>(d[1][grp >> 1], lo.z, lo.w, hi.z, hi.w, qb[grp][0], qb[grp][1]);
      }
      // x[i]: this lane's part of the score of token g + 8 i
      float x[4] = {start, start, start, start};
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int grp = min(2 * p + acc_group, G - 1);
        const uint4 w = *reinterpret_cast<const uint4*>(kt + kCodes + grp * 128 + g * 16);
        const uint32_t par[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int (&dd)[4] = d[i >> 1][p];
          const float dot = static_cast<float>(dd[2 * (i & 1)] + (dd[2 * (i & 1) + 1] << 8)) * qscale[p];
          const float step = bf16_low(par[i]);
          x[i] = fmaf(step, dot, fmaf(fmaf(kMiddle, step, bf16_high(par[i])), qsum[p], x[i]));
        }
      }
      // the four lanes of a row add up and lane j keeps token t = g + 8 j
      const float r0 = (j & 2 ? x[2] : x[0]) + __shfl_xor_sync(0xffffffffu, j & 2 ? x[0] : x[2], 2);
      const float r1 = (j & 2 ? x[3] : x[1]) + __shfl_xor_sync(0xffffffffu, j & 2 ? x[1] : x[3], 2);
      score[u] = (j & 1 ? r1 : r0) + __shfl_xor_sync(0xffffffffu, j & 1 ? r0 : r1, 1);
    }
    // ---- the steps and least values of the tokens that are there, and the weights' bytes
    // as they are where neither the maximum nor the fixed point has to move
    float pr[N];
    bool over = fresh;
    auto weigh = [&](int u) {
      pr[u] = in[u] ? exp2_fast(score[u]) : 0.0f;
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const float w = pr[u] * bf16_low(par[u][i]) * wup[i];
        over |= w >= 2147483648.0f;
        sh.weights[warp][u][i][t] = __float2uint_rn(w);
      }
    };
#pragma unroll
    for (int u = 0; u < N; ++u) {
      in[u] = (it + u) * 32 + t < end;
      over |= in[u] && score[u] > kKvqSlack;
#pragma unroll
      for (int i = 0; i < G; ++i)
        par[u][i] = in[u] ? *reinterpret_cast<const uint32_t*>(tile + u * kTileBytes + kTileBytes / 2 +
                                                               kCodes + i * 128 + lane * 4)
                          : 0;
      weigh(u);
    }
    // ---- softmax: m, the maximum that scores and weights refer to, is raised only
    // when a score passes it by kKvqSlack, the fixed points only when a weight times
    // its step passes them: one vote for all in most turns
    if (__any_sync(0xffffffffu, over)) {
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < N; ++u) top = fmaxf(top, in[u] ? score[u] : -INFINITY);
      top = warp_max(top);
      float raise = 0.0f, keep = 1.0f;
      if (top > 0.0f || (fresh && top > -INFINITY)) {
        const float old = m;
        m = old + top;
        // (2^20 and above, where a place of m is 1/8 and more: against this tile's top,
        // so that it weighs 1 whatever m was rounded to)
        raise = fabsf(m) < kKvqVast ? m - old : top;
        start = j & 1 ? -0.5f * m : 0.0f;
        keep = fresh ? 0.0f : exp2_fast(-raise);
        fresh = false;
        l *= keep;
#pragma unroll
        for (int i = 0; i < G; ++i) middle[i] *= keep;
#pragma unroll
        for (int p = 0; p < P; ++p) {
          o[p][0][0] *= keep;
          o[p][0][1] *= keep;
          o[p][1][0] *= keep;
          o[p][1][1] *= keep;
        }
      }
      // the fixed point of a group: its largest weight times step so far, as it stands
      // to m, lies in its upper half.  (By the largest step alone, a token of no weight
      // whose values are 10^5 times the others' would cost them their bits.)
      int e[G];
#pragma unroll
      for (int u = 0; u < N; ++u) {
        score[u] -= raise;
        pr[u] = in[u] ? exp2_fast(score[u]) : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < G; ++i) {
        float big = 0.0f;
#pragma unroll
        for (int u = 0; u < N; ++u) big = fmaxf(big, pr[u] * bf16_low(par[u][i]));  // (NaN counts as nothing)
        seen[i] = fmaxf(seen[i] * keep, __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big))));
        // weight times step < 2^(e - 126); below 2^-86 they lose precision
        e[i] = max(static_cast<int>(__float_as_uint(seen[i]) >> 23), 40);
        wup[i] = __uint_as_float(static_cast<uint32_t>(284 - e[i]) << 23);
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int ep = acc_group && 2 * p + 1 < G ? e[min(2 * p + 1, G - 1)] : e[2 * p];
        wdown[p] = __uint_as_float(static_cast<uint32_t>(ep - 30 - kShift + (j & 1) * 16) << 23);
      }
      if (fabsf(raise) > kKvqFar && fabsf(m) < kKvqVast && !again) {
        again = true;
        continue;
      }
#pragma unroll
      for (int u = 0; u < N; ++u) weigh(u);
    }
    again = false;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      l += pr[u];
#pragma unroll
      for (int i = 0; i < G; ++i)
        middle[i] = fmaf(pr[u], fmaf(kMiddle, bf16_low(par[u][i]), bf16_high(par[u][i])), middle[i]);
    }
    __syncwarp();
    // ---- values
#pragma unroll
    for (int p = 0; p < P; ++p) {
      int d[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const unsigned char* vt = tile + u * kTileBytes + kTileBytes / 2;
        const uint32_t* wp = sh.weights[warp][u][min(2 * p + col_group, G - 1)];
        const uint4 w0 = *reinterpret_cast<const uint4*>(wp + 4 * j);
        const uint4 w1 = *reinterpret_cast<const uint4*>(wp + 16 + 4 * j);
        const uint32_t b0 = gather_bytes(w0.x, w0.y, w0.z, w0.w, col_byte);
        const uint32_t b1 = gather_bytes(w1.x, w1.y, w1.z, w1.w, col_byte);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int grp = 2 * p + c;
          if (grp >= G) break;
          const uint32_t c0 = col_group == c ? b0 : 0, c1 = col_group == c ? b1 : 0;
          if (BITS == 4) {
            const uint4 w = *reinterpret_cast<const uint4*>(vt + grp * 512 + lane * 16);
            mma_s8_m16n8k32<false>(d[0], nibbles_low(w.x), nibbles_high(w.x), nibbles_low(w.y),
                                   nibbles_high(w.y), c0, c1);
            mma_s8_m16n8k32<false>(d[1], nibbles_low(w.z), nibbles_high(w.z), nibbles_low(w.w),
                                   nibbles_high(w.w), c0, c1);
          } else {
            const uint4 v0 = *reinterpret_cast<const uint4*>(vt + grp * 1024 + lane * 16);
            const uint4 v1 = *reinterpret_cast<const uint4*>(vt + grp * 1024 + 512 + lane * 16);
            mma_s8_m16n8k32<false>(d[0], v0.x, v0.y, v0.z, v0.w, c0, c1);
            mma_s8_m16n8k32<false>(d[1], v1.x, v1.y, v1.z, v1.w, c0, c1);
          }
        }
      }
      // (sums of N tiles: at most 2 * 32 * 128 * 255 * 257 < 2^31)
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int up = 0; up < 2; ++up)
          o[p][mb][up] = fmaf(static_cast<float>(d[mb][2 * up] + (d[mb][2 * up + 1] << 8)), wdown[p],
                              o[p][mb][up]);
    }
    __syncwarp();  // every lane has read the slot and the weights
    if (lane == 0 && it + kKvqSlots * N < last) fetch(it + kKvqSlots * N, slot);
    if (++slot == kKvqSlots) {
      slot = 0;
      phase ^= 1;
    }
    it += N;
  }

  // The next kernel (usually a push) may become resident now: earlier, its CTAs
  // take the registers that this one's last CTAs wait for (43.6 -> 42.3 us for
  // push and attention of 64 sequences x 2176 tokens).
  pdl_launch_dependents();
  // ---- the warps' parts
  l = warp_sum(l);
#pragma unroll
  for (int i = 0; i < G; ++i) middle[i] = warp_sum(middle[i]);
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int up = 0; up < 2; ++up) {
        const float v = o[p][mb][up] + __shfl_xor_sync(0xffffffffu, o[p][mb][up], 1);
        const float add = acc_group && 2 * p + 1 < G ? middle[min(2 * p + 1, G - 1)] : middle[2 * p];
        if (!(j & 1) && 2 * p + acc_group < G)
          sh.o[warp][(2 * p + acc_group) * 32 + mb * 16 + up * 8 + g] = v + add;
      }
  if (lane == 0) {
    sh.m[warp] = fresh ? -INFINITY : m;
    sh.l[warp] = l;
  }
  __syncthreads();
  float M = sh.m[0], L = 0.0f, f[W];
#pragma unroll
  for (int w = 1; w < W; ++w) M = fmaxf(M, sh.m[w]);
#pragma unroll
  for (int w = 0; w < W; ++w) {
    f[w] = part_factor(sh.m[w], sh.l[w], M);
    L = fmaf(f[w], sh.l[w], L);
  }
  // out[d] of the whole from the joined value of dim d and the sum L
  const int dim = a.layout.dim;
  auto finish = [&](auto value) {  // value(d) by whole warps; it may set M and L
    for (int d = threadIdx.x; d < G * 32; d += W * 32) {
      const float v = value(d);
      const bool bad = !(L > 0.0f && L < INFINITY) || !isfinite(M);
      if (bad && d == 0) flag(a.status, DEV_SOFTMAX);
      if (d < dim) a.out[row + d] = bad ? __uint_as_float(0x7FC00000u) : v / L;
    }
  };
  auto of_warps = [&](int d) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) v = fmaf(f[w], sh.o[w][d], v);
    return v;
  };
  if (splits == 1) {
    finish(of_warps);
    return;
  }
  // ---- the CTAs of a cluster, by its first
  for (int d = threadIdx.x; d < G * 32; d += W * 32) sh.o[0][d] = of_warps(d);  // (own element)
  if (threadIdx.x == 0) {
    sh.cta_m = M;
    sh.cta_l = L;
  }
  cluster_arrive();
  cluster_wait();
  if (rank == 0) {
    // lane r weighs part r; a part's values are loaded before its weight is known
    float part;
    auto weigh = [&](float pm, float pl) {
      M = warp_max(pm);
      part = part_factor(pm, pl, M);
      L = warp_sum(part * pl);
    };
    const bool mine = lane < splits;
    weigh(mine ? cluster_load(&sh.cta_m, lane) : -INFINITY, mine ? cluster_load(&sh.cta_l, lane) : 0.0f);
    auto of_cluster = [&](int d) {
      float v[kKvqCluster], sum = 0.0f;
#pragma unroll
      for (int r = 0; r < kKvqCluster; ++r) v[r] = r < splits ? cluster_load(&sh.o[0][d], r) : 0.0f;
#pragma unroll
      for (int r = 0; r < kKvqCluster; ++r) sum = fmaf(__shfl_sync(0xffffffffu, part, r), v[r], sum);
      return sum;
    };
    if (a.parts == 1) {
      finish(of_cluster);
    } else {
      // ---- the clusters of a head, by the one that ends last, in their order
      const int unit = b * a.layout.heads + h, stride = dim + 2;
      float* all = a.partial + static_cast<long long>(unit) * a.parts * stride;
      float* own = all + share / splits * stride;
      for (int d = threadIdx.x; d < G * 32; d += W * 32) {
        const float v = of_cluster(d);
        if (d < dim) own[2 + d] = v;
      }
      if (threadIdx.x == 0) {
        own[0] = M;
        own[1] = L;
      }
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) sh.turn = atomicAdd(a.tickets + unit, 1);
      __syncthreads();
      if (sh.turn == a.parts - 1) {
        __threadfence();
        if (threadIdx.x == 0) a.tickets[unit] = 0;  // for the next launch
        const bool there = lane < a.parts;
        const float pm = there ? __ldcg(all + lane * stride) : -INFINITY;
        const float pl = there ? __ldcg(all + lane * stride + 1) : 0.0f;
        bool weighed = false;
        auto of_parts = [&](int d) {
          float v[kKvqMaxParts], sum = 0.0f;
#pragma unroll
          for (int r = 0; r < kKvqMaxParts; ++r)
            v[r] = r < a.parts && d < dim ? __ldcg(all + r * stride + 2 + d) : 0.0f;
          if (!weighed) weigh(pm, pl);
          weighed = true;
#pragma unroll
          for (int r = 0; r < kKvqMaxParts; ++r) sum = fmaf(__shfl_sync(0xffffffffu, part, r), v[r], sum);
          return sum;
        };
        finish(of_parts);
      }
    }
  }
  cluster_arrive();  // no CTA leaves while its part may still be read
  cluster_wait();
}

template <int G, int BITS>
static cudaError_t launch_kvq_attention_t(KvqAttnArgs a, int batch, cudaStream_t st) {
  using Shared = KvqShared<G, BITS>;
  constexpr size_t smem = sizeof(Shared);
  static_assert(smem <= 227 * 1024, "shared memory of a CTA");
  static PerDeviceOnce configured;
  configured.run([] {
    cudaFuncSetAttribute(kvq_attention_kernel<G, BITS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         static_cast<int>(smem));
  });
  // Every CTA resident at once where the heads are few: clusters of up to eight
  // while the warps of a head outnumber no tiles of a full cache, then several
  // clusters per head while every warp keeps 4 tiles (one sequence of 32,768 tokens,
  // 10 heads: 32 us without the second step, 17.9 with it, 22.7 where warps may keep
  // fewer tiles and the CTAs no longer fit at once).
  constexpr int W = Shared::W;
  const long long heads = static_cast<long long>(batch) * a.layout.heads;
  constexpr int kPerSm = 227 * 1024 / (smem + 1024);
  const long long slots = static_cast<long long>(a.sms) * (kPerSm < kKvqCtasPerSm ? kPerSm : kKvqCtasPerSm);
  a.splits = a.parts = 1;
  while (a.splits < kKvqCluster && 2 * heads * a.splits <= slots && a.layout.tiles > a.splits * W)
    a.splits *= 2;
  if (a.splits > 1) {
    const long long most = slots / (heads * a.splits), fed = a.layout.tiles / (a.splits * W * 4);
    const long long parts = most < fed ? most : fed;
    a.parts = parts < 1 ? 1 : parts > kKvqMaxParts ? kKvqMaxParts : static_cast<int>(parts);
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(a.splits), 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.layout.heads * a.splits * a.parts, batch);
  cfg.blockDim = dim3(W * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kvq_attention_kernel<G, BITS>, a);
  if (e != cudaSuccess) {  // without the early start
    cudaGetLastError();
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kvq_attention_kernel<G, BITS>, a);
  }
  return e;
}

template <int BITS>
static cudaError_t launch_kvq_attention_b(const KvqAttnArgs& a, int batch, cudaStream_t st) {
  switch (a.layout.groups) {
    case 1: return launch_kvq_attention_t<1, BITS>(a, batch, st);
    case 2: return launch_kvq_attention_t<2, BITS>(a, batch, st);
    case 3: return launch_kvq_attention_t<3, BITS>(a, batch, st);
    case 4: return launch_kvq_attention_t<4, BITS>(a, batch, st);
    case 5: return launch_kvq_attention_t<5, BITS>(a, batch, st);
    case 6: return launch_kvq_attention_t<6, BITS>(a, batch, st);
    case 7: return launch_kvq_attention_t<7, BITS>(a, batch, st);
    case 8: return launch_kvq_attention_t<8, BITS>(a, batch, st);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_kvq_attention(const KvqAttnArgs& a, int batch, cudaStream_t st) {
  return a.layout.bits == 4 ? launch_kvq_attention_b<4>(a, batch, st)
                            : launch_kvq_attention_b<8>(a, batch, st);
}

}  // namespace uocr
