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
// One query per (head, sequence) over the tiles of its cache.  The codes go to
// the matrix unit as they are (u8, m16n8k32), the query and the softmax weights
// as fixed-point numbers cut into bytes, one byte per column of the 8-wide
// operand, so that every product is exact and nothing is dequantised:
//
//   scores:  rows = 16 tokens, k = the 32 dims of a group, columns = the four
//            signed bytes of q 2^a (|q 2^a| < 2^30, a by the group's largest |q|);
//            q . c = sum_b 256^b D_b, then s (q . c) + m sum(q) per group;
//   values:  rows = 16 dims, k = the tile's 32 tokens, columns = the four bytes
//            of p_t s_t 2^a (< 2^31, a by the largest s so far);
//            o += 2^-a sum_b 256^b D_b, and p_t m_t is summed apart.
//
// Two neighbouring groups share an accumulator: a group's operand has its bytes
// in its four columns and zeros in the other group's four.  Fixed point loses
// less than a float does: 2^-31 of the group's largest |q|, 2^-32 of the
// largest step, against a float's 2^-24 of each term.
//
// A tile is one bulk copy.  Every warp has a ring of its own, takes a run of
// neighbouring tiles, and keeps its own maximum, sum and weighted values, so the
// loop has no barrier but the ring's.  The warps' parts are joined in shared
// memory, the CTAs' of one head through distributed shared memory: one launch,
// no workspace.
constexpr int kKvqWarps = 4;
constexpr float kLog2e = 1.44269504f;

__host__ __device__ constexpr int kvq_tile_bytes(int groups, int bits) {
  return 2 * groups * (512 * (bits / 4) + 128);
}
// Ring slots per warp: about 20 KB, two at least, eight at most.
__host__ __device__ constexpr int kvq_slots(int groups, int bits) {
  const int n = 20480 / kvq_tile_bytes(groups, bits);
  return n < 2 ? 2 : n > 8 ? 8 : n;
}

template <int G, int BITS>
struct KvqShared {
  static constexpr int kSlots = kvq_slots(G, BITS);
  alignas(128) unsigned char ring[kKvqWarps][kSlots][kvq_tile_bytes(G, BITS)];
  alignas(16) uint32_t weights[kKvqWarps][G][32];
  uint64_t full[kKvqWarps][kSlots];
  float o[kKvqWarps][G * 32];  // weighted values per warp; the CTA's in [0]
  float m[kKvqWarps], l[kKvqWarps];
  float cta_m, cta_l;
};

// u8 rows times signed (SIGNED) or unsigned columns, 32-bit sums.
template <bool SIGNED>
__device__ __forceinline__ void mma_u8_m16n8k32(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                                uint32_t a3, uint32_t b0, uint32_t b1) {
  if (SIGNED)
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

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
  return m == -INFINITY && l == 0.0f ? 0.0f : exp2_fast((m - M) * kLog2e);
}

template <int G, int BITS>
__global__ void __launch_bounds__(kKvqWarps * 32) kvq_attention_kernel(const KvqAttnArgs a) {
  constexpr int P = (G + 1) / 2;  // accumulators: pairs of groups
  using Shared = KvqShared<G, BITS>;
  constexpr int kSlots = Shared::kSlots, kTileBytes = kvq_tile_bytes(G, BITS);
  constexpr int kCodes = G * 512 * (BITS / 4);
  extern __shared__ __align__(128) unsigned char kvq_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(kvq_raw);
  pdl_launch_dependents();  // launched as a programmatic dependent (launch_dependent):
  pdl_wait_prior_grids();   // nothing is touched before the previous kernel completes
  const int splits = a.splits;
  const int h = blockIdx.x / splits, rank = blockIdx.x % splits, b = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  const int T = kvq_tokens(a.state, b, a.window);
  if (T <= 0) {  // the same for every CTA of the cluster
    if (threadIdx.x == 0 && rank == 0) flag(a.status, DEV_CACHE);
    return;
  }
  const int tiles = (T + 31) >> 5, workers = splits * kKvqWarps, me = rank * kKvqWarps + warp;
  const int first = static_cast<int>(static_cast<long long>(tiles) * me / workers);
  const int last = static_cast<int>(static_cast<long long>(tiles) * (me + 1) / workers);
  const unsigned char* head =
      a.data + (static_cast<long long>(b) * a.layout.heads + h) * a.layout.tiles * kTileBytes;
  if (lane == 0) {
    for (int i = 0; i < kSlots; ++i) mbar_init(&sh.full[warp][i], 1);
    fence_mbar_init();
    for (int i = 0; i < kSlots && first + i < last; ++i) {
      mbar_arrive_expect_tx(&sh.full[warp][i], kTileBytes);
      bulk_g2s(sh.ring[warp][i], head + static_cast<long long>(first + i) * kTileBytes, kTileBytes,
               &sh.full[warp][i]);
    }
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
    float v[8], big = 0.0f, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = grp * 32 + (i >> 2) * 16 + 4 * j + (i & 3);
      v[i] = d < a.layout.dim ? __ldg(a.q + row + d) : 0.0f;
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
    // bytes) and, once, the sum; NaN and infinities of q reach the scores by it
    const int ea = __shfl_sync(0xffffffffu, e, acc_group * 16);
    const float sa = __shfl_sync(0xffffffffu, sum, acc_group * 16);
    const bool real = 2 * p + acc_group < G;
    qscale[p] = real ? __uint_as_float(static_cast<uint32_t>(min(ea, 254) - 29 + (j & 1) * 16) << 23) : 0.0f;
    qsum[p] = real && !(j & 1) ? sa : 0.0f;
  }

  float m = -INFINITY, l = 0.0f, least[G], o[P][2][2];
  uint32_t bound[G];    // largest step so far per group, as bf16 bits
  float wup[G], wdown[P];
#pragma unroll
  for (int i = 0; i < G; ++i) {
    least[i] = 0.0f;
    bound[i] = 0;
    wup[i] = 0.0f;
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
    wdown[p] = 0.0f;
    o[p][0][0] = o[p][0][1] = o[p][1][0] = o[p][1][1] = 0.0f;
  }

  for (int it = first, slot = 0, phase = 0; it < last; ++it) {
    if (!__all_sync(0xffffffffu, mbar_wait_try(&sh.full[warp][slot], phase, a.status))) {
      // (a safety net: flagged) copies in flight land before the CTA ends
      for (int i = 1; i < kSlots && it + i < last; ++i) {
        if (++slot == kSlots) {
          slot = 0;
          phase ^= 1;
        }
        mbar_wait_try(&sh.full[warp][slot], phase, a.status);
      }
      break;
    }
    const unsigned char* tile = sh.ring[warp][slot];
    // ---- scores: x[i] is this lane's part of the score of token g + 8 i
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    {
      int d[2][P][4];
#pragma unroll
      for (int i = 0; i < 2 * P * 4; ++i) (&d[0][0][0])[i] = 0;
#pragma unroll
      for (int grp = 0; grp < G; ++grp) {
        uint4 lo, hi;
        if (BITS == 4) {
          const uint4 w = *reinterpret_cast<const uint4*>(tile + grp * 512 + lane * 16);
          lo = make_uint4(w.x & 0x0F0F0F0Fu, w.y & 0x0F0F0F0Fu, w.z & 0x0F0F0F0Fu, w.w & 0x0F0F0F0Fu);
          hi = make_uint4((w.x >> 4) & 0x0F0F0F0Fu, (w.y >> 4) & 0x0F0F0F0Fu,
                          (w.z >> 4) & 0x0F0F0F0Fu, (w.w >> 4) & 0x0F0F0F0Fu);
        } else {
          lo = *reinterpret_cast<const uint4*>(tile + grp * 1024 + lane * 16);
          hi = *reinterpret_cast<const uint4*>(tile + grp * 1024 + 512 + lane * 16);
        }
        mma_u8_m16n8k32<true>(d[0][grp >> 1], lo.x, lo.y, hi.x, hi.y, qb[grp][0], qb[grp][1]);
        mma_u8_m16n8k32<true>(d[1][grp >> 1], lo.z, lo.w, hi.z, hi.w, qb[grp][0], qb[grp][1]);
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int grp = min(2 * p + acc_group, G - 1);
        const uint4 w = *reinterpret_cast<const uint4*>(tile + kCodes + grp * 128 + g * 16);
        const uint32_t par[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int (&dd)[4] = d[i >> 1][p];
          const float dot = static_cast<float>(dd[2 * (i & 1)] + (dd[2 * (i & 1) + 1] << 8)) * qscale[p];
          x[i] = fmaf(bf16_low(par[i]), dot, fmaf(bf16_high(par[i]), qsum[p], x[i]));
        }
      }
    }
    // the four lanes of a row add up and lane j keeps token t = g + 8 j
    const float r0 = (j & 2 ? x[2] : x[0]) + __shfl_xor_sync(0xffffffffu, j & 2 ? x[0] : x[2], 2);
    const float r1 = (j & 2 ? x[3] : x[1]) + __shfl_xor_sync(0xffffffffu, j & 2 ? x[1] : x[3], 2);
    const float score =
        ((j & 1 ? r1 : r0) + __shfl_xor_sync(0xffffffffu, j & 1 ? r0 : r1, 1)) * a.scale;
    const int t = g + 8 * j;
    const bool in = it * 32 + t < T;
    // ---- softmax
    const float top = warp_max(in ? score : -INFINITY);
    if (top > m) {
      const float keep = exp2_fast((m - top) * kLog2e);
      m = top;
      l *= keep;
#pragma unroll
      for (int i = 0; i < G; ++i) least[i] *= keep;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        o[p][0][0] *= keep;
        o[p][0][1] *= keep;
        o[p][1][0] *= keep;
        o[p][1][1] *= keep;
      }
    }
    const float pr = in ? exp2_fast((score - m) * kLog2e) : 0.0f;
    l += pr;
    // ---- the weights' bytes
    const unsigned char* vt = tile + kTileBytes / 2;
    uint32_t par[G];
    bool over = false;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      // a token that is not there: nothing of what its slot holds
      par[i] = in ? *reinterpret_cast<const uint32_t*>(vt + kCodes + i * 128 + lane * 4) : 0;
      over |= (par[i] & 0xFFFFu) > bound[i];
    }
    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
      for (int i = 0; i < G; ++i) {
        bound[i] = max(bound[i], __reduce_max_sync(0xffffffffu, par[i] & 0xFFFFu));
        // step < 2^(e - 126); steps below 2^-86 lose precision
        const uint32_t e = max(bound[i] >> 7, 40u);
        wup[i] = __uint_as_float((284u - e) << 23);
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const uint32_t bd = acc_group && 2 * p + 1 < G ? bound[min(2 * p + 1, G - 1)] : bound[2 * p];
        wdown[p] = __uint_as_float((max(bd >> 7, 40u) - 30u + (j & 1) * 16u) << 23);
      }
    }
#pragma unroll
    for (int i = 0; i < G; ++i) {
      least[i] = fmaf(pr, bf16_high(par[i]), least[i]);
      sh.weights[warp][i][t] = __float2uint_rn(pr * (bf16_low(par[i]) * wup[i]));
    }
    __syncwarp();
    // ---- values
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint32_t* wp = sh.weights[warp][min(2 * p + col_group, G - 1)];
      const uint4 w0 = *reinterpret_cast<const uint4*>(wp + 4 * j);
      const uint4 w1 = *reinterpret_cast<const uint4*>(wp + 16 + 4 * j);
      const uint32_t b0 = gather_bytes(w0.x, w0.y, w0.z, w0.w, col_byte);
      const uint32_t b1 = gather_bytes(w1.x, w1.y, w1.z, w1.w, col_byte);
      int d[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int grp = 2 * p + c;
        if (grp >= G) break;
        const uint32_t c0 = col_group == c ? b0 : 0, c1 = col_group == c ? b1 : 0;
        if (BITS == 4) {
          const uint4 w = *reinterpret_cast<const uint4*>(vt + grp * 512 + lane * 16);
          mma_u8_m16n8k32<false>(d[0], w.x & 0x0F0F0F0Fu, (w.x >> 4) & 0x0F0F0F0Fu, w.y & 0x0F0F0F0Fu,
                                 (w.y >> 4) & 0x0F0F0F0Fu, c0, c1);
          mma_u8_m16n8k32<false>(d[1], w.z & 0x0F0F0F0Fu, (w.z >> 4) & 0x0F0F0F0Fu, w.w & 0x0F0F0F0Fu,
                                 (w.w >> 4) & 0x0F0F0F0Fu, c0, c1);
        } else {
          const uint4 v0 = *reinterpret_cast<const uint4*>(vt + grp * 1024 + lane * 16);
          const uint4 v1 = *reinterpret_cast<const uint4*>(vt + grp * 1024 + 512 + lane * 16);
          mma_u8_m16n8k32<false>(d[0], v0.x, v0.y, v0.z, v0.w, c0, c1);
          mma_u8_m16n8k32<false>(d[1], v1.x, v1.y, v1.z, v1.w, c0, c1);
        }
      }
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int up = 0; up < 2; ++up)
          o[p][mb][up] = fmaf(static_cast<float>(d[mb][2 * up] + (d[mb][2 * up + 1] << 8)), wdown[p],
                              o[p][mb][up]);
    }
    __syncwarp();  // every lane has read the slot and the weights
    if (lane == 0 && it + kSlots < last) {
      mbar_arrive_expect_tx(&sh.full[warp][slot], kTileBytes);
      bulk_g2s(sh.ring[warp][slot], head + static_cast<long long>(it + kSlots) * kTileBytes, kTileBytes,
               &sh.full[warp][slot]);
    }
    if (++slot == kSlots) {
      slot = 0;
      phase ^= 1;
    }
  }

  // ---- the warps' parts
  l = warp_sum(l);
#pragma unroll
  for (int i = 0; i < G; ++i) least[i] = warp_sum(least[i]);
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int up = 0; up < 2; ++up) {
        const float v = o[p][mb][up] + __shfl_xor_sync(0xffffffffu, o[p][mb][up], 1);
        const float add = acc_group && 2 * p + 1 < G ? least[min(2 * p + 1, G - 1)] : least[2 * p];
        if (!(j & 1) && 2 * p + acc_group < G)
          sh.o[warp][(2 * p + acc_group) * 32 + mb * 16 + up * 8 + g] = v + add;
      }
  if (lane == 0) {
    sh.m[warp] = m;
    sh.l[warp] = l;
  }
  __syncthreads();
  float M = sh.m[0], L = 0.0f, f[kKvqWarps];
#pragma unroll
  for (int w = 1; w < kKvqWarps; ++w) M = fmaxf(M, sh.m[w]);
#pragma unroll
  for (int w = 0; w < kKvqWarps; ++w) {
    f[w] = part_factor(sh.m[w], sh.l[w], M);
    L = fmaf(f[w], sh.l[w], L);
  }
  if (splits > 1) {
    for (int d = threadIdx.x; d < G * 32; d += kKvqWarps * 32) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kKvqWarps; ++w) v = fmaf(f[w], sh.o[w][d], v);
      sh.o[0][d] = v;  // read and written by this thread alone
    }
    if (threadIdx.x == 0) {
      sh.cta_m = M;
      sh.cta_l = L;
    }
    cluster_arrive();
    cluster_wait();
    float cm[16], cf[16];
    M = -INFINITY;
    for (int r = 0; r < splits; ++r) M = fmaxf(M, cm[r] = cluster_load(&sh.cta_m, r));
    L = 0.0f;
    for (int r = 0; r < splits; ++r) {
      const float cl = cluster_load(&sh.cta_l, r);
      cf[r] = part_factor(cm[r], cl, M);
      L = fmaf(cf[r], cl, L);
    }
    const bool bad = !(L > 0.0f && L < INFINITY) || !isfinite(M);
    for (int d = rank * kKvqWarps * 32 + threadIdx.x; d < a.layout.dim; d += splits * kKvqWarps * 32) {
      float v = 0.0f;
      for (int r = 0; r < splits; ++r) v = fmaf(cf[r], cluster_load(&sh.o[0][d], r), v);
      a.out[row + d] = bad ? __uint_as_float(0x7FC00000u) : v / L;
    }
    if (bad && rank == 0 && threadIdx.x == 0) flag(a.status, DEV_SOFTMAX);
    cluster_arrive();  // no CTA leaves while its part may still be read
    cluster_wait();
    return;
  }
  const bool bad = !(L > 0.0f && L < INFINITY) || !isfinite(M);
  if (bad && threadIdx.x == 0) flag(a.status, DEV_SOFTMAX);
  for (int d = threadIdx.x; d < a.layout.dim; d += kKvqWarps * 32) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kKvqWarps; ++w) v = fmaf(f[w], sh.o[w][d], v);
    a.out[row + d] = bad ? __uint_as_float(0x7FC00000u) : v / L;
  }
}

template <int G, int BITS>
static cudaError_t launch_kvq_attention_t(const KvqAttnArgs& a, int batch, cudaStream_t st) {
  constexpr size_t smem = sizeof(KvqShared<G, BITS>);
  static_assert(smem <= 227 * 1024, "shared memory of a CTA");
  static PerDeviceOnce configured;
  configured.run([] {
    cudaFuncSetAttribute(kvq_attention_kernel<G, BITS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         static_cast<int>(smem));
  });
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(a.splits), 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.layout.heads * a.splits, batch);
  cfg.blockDim = dim3(kKvqWarps * 32);
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

cudaError_t launch_kvq_attention(KvqAttnArgs a, int batch, cudaStream_t st) {
  // CTAs per head: enough for two per SM, at most a portable cluster, and no
  // more than leave every warp a tile of a full cache
  const long long heads = static_cast<long long>(batch) * a.layout.heads;
  a.splits = 1;
  while (a.splits < 8 && heads * a.splits < 2LL * a.sms &&
         a.layout.tiles > static_cast<long long>(a.splits) * kKvqWarps)
    a.splits *= 2;
  return a.layout.bits == 4 ? launch_kvq_attention_b<4>(a, batch, st)
                            : launch_kvq_attention_b<8>(a, batch, st);
}

}  // namespace uocr
