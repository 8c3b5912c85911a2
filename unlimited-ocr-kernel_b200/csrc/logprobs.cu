// logprobs.cu — log probabilities of given tokens, entropies and the most
// probable alternatives of rows of logits.
//
// Per row x of V logits, M = max x at its lowest index i*, z_i = x_i - M <= 0:
//   S' = sum_{i != i*} e^{z_i},  log sum e^{z_i} = log1p(S'),
//   log p(t) = z_t - log1p(S'),  H = log1p(S') + (sum e^{z_i} (-z_i)) / (1 + S').
// Leaving the maximum's own 1 out of the sum keeps the log probability of a
// nearly certain token and a nearly zero entropy exact to a float's relative
// precision, and both terms of H are >= 0, so nothing cancels.
#include <cuda_runtime.h>

#include "common.cuh"
#include "kernels.h"

namespace uocr {

constexpr int kLpThreads = 256;

// Orders logits: larger first, then the lower index.  -0 and +0 are equal.
__device__ __forceinline__ unsigned long long lp_key(float x, int i) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  const uint32_t o = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (static_cast<unsigned long long>(o) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ int lp_index(unsigned long long key) {
  return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key));
}

__device__ __forceinline__ unsigned long long lp_block_max(unsigned long long v,
                                                           unsigned long long* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int w = 0; w < kLpThreads / 32; ++w) v = red[w] > v ? red[w] : v;
  return v;
}

__device__ __forceinline__ float lp_block_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int w = 0; w < kLpThreads / 32; ++w) v += red[w];
  return v;
}

__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(const LogprobArgs a) {
  __shared__ unsigned long long kred[kLpThreads / 32];
  __shared__ float fred[kLpThreads / 32];
  const int row = blockIdx.x;
  const float* x = a.logits + row * a.ld;
  const float nan = __uint_as_float(0x7FC00000u);
  unsigned long long best = 0;
  bool bad = false;
  for (int i = threadIdx.x; i < a.vocab; i += kLpThreads) {
    bad |= !(x[i] < INFINITY);  // NaN or +inf
    const unsigned long long k = lp_key(x[i], i);
    best = k > best ? k : best;
  }
  bad = __syncthreads_or(bad);
  best = lp_block_max(best, kred);
  const int top = lp_index(best);
  const float m = bad ? 0.0f : x[top];
  bad |= m == -INFINITY;
  float s = 0.0f, w = 0.0f;
  for (int i = threadIdx.x; i < a.vocab && !bad; i += kLpThreads)
    if (i != top) {
      const float z = x[i] - m, e = expf(z);
      s += e;
      w += e * fmaxf(z, -1000.0f);
    }
  s = lp_block_sum(s, fred);
  w = lp_block_sum(w, fred);
  const float lse = log1pf(s);
  if (threadIdx.x == 0) {
    if (bad) flag(a.status, DEV_SOFTMAX);
    if (a.entropy) a.entropy[row] = bad ? nan : lse - w / (1.0f + s);
    if (a.logprob) {
      const long long t = a.tokens[row];
      if (t >= a.vocab) flag(a.status, DEV_TOKEN);
      a.logprob[row] = bad || t >= a.vocab ? nan : t < 0 ? 0.0f : (x[t] - m) - lse;
    }
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < a.top_k; ++j) {
    unsigned long long next = 0;
    for (int i = threadIdx.x; i < a.vocab && !bad; i += kLpThreads) {
      const unsigned long long k = lp_key(x[i], i);
      if (k < last && k > next) next = k;
    }
    last = lp_block_max(next, kred);
    if (threadIdx.x == 0) {
      const int i = lp_index(last);
      const long long o = static_cast<long long>(row) * a.top_k + j;
      a.top_ids[o] = bad ? -1 : i;
      a.top_logprobs[o] = bad ? nan : (x[i] - m) - lse;
    }
  }
}

cudaError_t launch_token_logprobs(const LogprobArgs& a, int rows, int sms, cudaStream_t st) {
  token_logprobs_kernel<<<rows, kLpThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace uocr
