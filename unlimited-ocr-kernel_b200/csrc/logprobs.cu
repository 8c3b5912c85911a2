// logprobs.cu — log probabilities of given tokens, entropies and the most
// probable alternatives of rows of logits.
//
// Per row x of V logits, M = max x, taken out of the sum once (n elements have
// it), z_i = x_i - M <= 0:
//   S' = sum_{z < 0} e^{z_i} + (n - 1),  log sum e^{z_i} = log1p(S'),
//   log p(t) = z_t - log1p(S'),  H = log1p(S') + (sum e^{z_i} (-z_i)) / (1 + S').
// Leaving the maximum's own 1 out of the sum keeps the log probability of a
// nearly certain token and a nearly zero entropy exact to a float's relative
// precision, and both terms of H are >= 0, so nothing cancels.
//
// One pass: every thread keeps the maximum of what it has seen, the sums that
// refer to it, and rescales them once per 16 elements.  The alternatives are
// those of a short list of candidates per CTA: an element enters it when its
// key (logit, then lower index) reaches the k-th best one known.  A first bound
// comes from the threads' maxima (k of them reach it, so k elements do); the
// list is cut back to its k best, in order, whenever it grows, which raises the
// bound.  A row is spread over a cluster of CTAs where the rows are few; the
// CTAs' sums and lists are joined through distributed shared memory.
#include <cuda_runtime.h>

#include "common.cuh"
#include "kernels.h"

namespace uocr {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpVec = 4;                    // 16-byte loads per thread and segment
constexpr int kLpPer = 4 * kLpVec;           // elements per thread and segment
constexpr int kLpSegment = kLpThreads * kLpVec;  // 16-byte vectors
constexpr int kLpCluster = 8;                // most CTAs per row (portable)
// Candidates: at most kLpCut stay after a cut, kLogprobMaxTop threads' elements
// join by the exact bound.
constexpr int kLpList = 1024;
constexpr int kLpCut = kLpList - kLogprobMaxTop * kLpPer;
constexpr float kLpLog2e = 1.44269504f;

using LpKey = unsigned long long;

// Orders logits: larger first, then the lower index.  -0 and +0 are equal.
__device__ __forceinline__ uint32_t lp_order(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ LpKey lp_key(float x, int i) {
  return (static_cast<LpKey>(lp_order(x)) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ int lp_index(LpKey key) {
  return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(key));
}
__device__ __forceinline__ float lp_logit(uint32_t order) {
  return __uint_as_float(order & 0x80000000u ? order & 0x7FFFFFFFu : ~order);
}

__device__ __forceinline__ float lp_exp2(float x) {  // 2 ulp
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct alignas(16) LpShared {
  LpKey list[2][kLpList];
  LpKey best[kLpCluster * kLogprobMaxTop];  // the CTA's best; the row's parts in the first CTA
  float m[kLpWarps], s[kLpWarps], w[kLpWarps], n[kLpWarps];
  float part[4];                   // the CTA's {M, S, W, n}
  uint32_t bound[kLpWarps];
  int count[2];
  LpKey floor;
};

// The k best of list[from][0, n), in order, into dst; the k-th best (0 while
// there are fewer) is the new floor.  All threads; a barrier before and after.
__device__ __forceinline__ void lp_cut(LpShared& sh, const LpKey* src, int n, int k, LpKey* dst) {
  for (int i = threadIdx.x; i < n; i += kLpThreads) {
    const LpKey mine = src[i];
    int rank = 0;
    int c = 0;
    for (; c + 2 <= n; c += 2) {
      const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(src + c);
      rank += (o.x > mine) + (o.y > mine);
    }
    if (c < n) rank += src[c] > mine;
    if (rank < k) dst[rank] = mine;
    if (rank == k - 1) sh.floor = mine;
  }
}

__device__ __forceinline__ uint32_t lp_mapped(const void* p, uint32_t rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
  return at;
}
__device__ __forceinline__ float lp_remote(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(lp_mapped(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ LpKey lp_remote(const LpKey* p, uint32_t rank) {
  LpKey v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(lp_mapped(p, rank)) : "memory");
  return v;
}

// Sums {S, W, n} that refer to a maximum m, as they stand to M >= m.
__device__ __forceinline__ void lp_refer(float m, float M, float& s, float& w, float& n) {
  if (m == M) return;
  const float d = fmaxf(m - M, -1000.0f), f = lp_exp2(d * kLpLog2e), all = s + n;
  w = f * fmaf(d, all, w);
  s = f * all;
  n = 0.0f;
}

template <bool TOP>
__global__ void __launch_bounds__(kLpThreads, 4) token_logprobs_kernel(const LogprobArgs a) {
  __shared__ LpShared sh;
  const int splits = a.splits, rank = blockIdx.x % splits, row = blockIdx.x / splits;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, k = a.top_k;
  const float* x = a.logits + row * a.ld;
  long long token = -1;
  float token_logit = 0.0f;
  if (a.tokens && rank == 0 && tid == 0) {
    token = a.tokens[row];
    if (token >= 0 && token < a.vocab) token_logit = __ldg(x + token);
  }
  // 16-byte vectors from the boundary at or before the row's first element, of
  // which `skip` elements are not the row's
  const int skip = static_cast<int>((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
  const float* base = x - skip;
  const long long end = static_cast<long long>(a.vocab) + skip;  // in elements of base
  const int vecs = static_cast<int>((end + 3) >> 2);
  const int first = static_cast<int>(static_cast<long long>(vecs) * rank / splits);
  const int last = static_cast<int>(static_cast<long long>(vecs) * (rank + 1) / splits);
  auto load = [&](int seg, float (&v)[kLpPer]) {
#pragma unroll
    for (int r = 0; r < kLpVec; ++r) {
      const int i = seg + r * kLpThreads + tid;
      if (i < last && (i > 0 || skip == 0) && 4LL * i + 4 <= end) {
        const float4 q = __ldcs(reinterpret_cast<const float4*>(base) + i);
        v[4 * r] = q.x;
        v[4 * r + 1] = q.y;
        v[4 * r + 2] = q.z;
        v[4 * r + 3] = q.w;
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const long long e = 4LL * i + c;
          v[4 * r + c] = i < last && e >= skip && e < end ? __ldcs(base + e) : -INFINITY;
        }
      }
    }
  };
  if (TOP) {
    if (tid < 2) sh.count[tid] = 0;
    if (tid == 0) sh.floor = 0;
    __syncthreads();
  }
  float m = -INFINITY, s = 0.0f, w = 0.0f, n = 0.0f;
  int cur = 0;  // the list in use
  float v[kLpPer];
  load(first, v);
  for (int seg = first; seg < last; seg += kLpSegment) {
    float next[kLpPer];
    if (seg + kLpSegment < last) load(seg + kLpSegment, next);
    float mx = v[0];
#pragma unroll
    for (int i = 1; i < kLpPer; ++i) mx = fmaxf(mx, v[i]);
    if (mx > m) {
      lp_refer(m, mx, s, w, n);
      m = mx;
    }
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < kLpPer; ++i) {
      const float z = v[i] - ref, e = lp_exp2(z * kLpLog2e);
      if (z != 0.0f) s += e;  // NaN stays in the sum
      else n += 1.0f;
      w = fmaf(e, fmaxf(z, -1000.0f), w);
    }
    if (TOP) {
      // the candidates of this segment
      LpKey floor = sh.floor;
      auto hits = [&] { return lp_order(mx) >= static_cast<uint32_t>(floor >> 32) && mx >= -INFINITY; };
      // key of v[i], 0 where the segment has run out of this CTA's elements
      auto key_of = [&](int i) {
        const int at = seg + (i >> 2) * kLpThreads + tid, e = 4 * at + (i & 3) - skip;
        return at < last && e >= 0 && e < a.vocab && !isnan(v[i]) ? lp_key(v[i], e) : 0;
      };
      const int before = sh.count[cur];  // (read ahead of the barrier: elements join behind it)
      int threads = __syncthreads_count(hits());
      if (threads) {
        if (before + threads * kLpPer > kLpList) {
          // a bound that k threads' maxima reach: the r-th best of every warp
          uint32_t o = lp_order(mx), nth = 0;
          for (int r = 0; r < (k + kLpWarps - 1) / kLpWarps; ++r) {
            nth = __reduce_max_sync(0xffffffffu, o);
            const unsigned who = __ballot_sync(0xffffffffu, o == nth);
            if (lane == __ffs(who) - 1) o = 0;
          }
          if (lane == 0) sh.bound[warp] = nth;
          __syncthreads();
          uint32_t low = sh.bound[0];
#pragma unroll
          for (int i = 1; i < kLpWarps; ++i) low = min(low, sh.bound[i]);
          const LpKey at_least = static_cast<LpKey>(low) << 32;
          floor = at_least > floor ? at_least : floor;
          threads = __syncthreads_count(hits());
        }
        bool joins;
        if (before + threads * kLpPer > kLpList) {
          // still too many, as equal logits can be: the exact k-th best of the
          // threads' best keys, which only k threads reach
          if (before > kLpCut) {  // room first
            lp_cut(sh, sh.list[cur], before, k, sh.list[cur ^ 1]);
            __syncthreads();
            if (tid == 0) sh.count[cur ^ 1] = k;
            cur ^= 1;
            __syncthreads();
          }
          LpKey best = 0;
#pragma unroll
          for (int i = 0; i < kLpPer; ++i) {
            const LpKey key = key_of(i);
            best = key > best ? key : best;
          }
          LpKey* keys = sh.list[cur ^ 1];
          keys[tid] = best;
          __syncthreads();
          int above = 0;
          for (int c = 0; c < kLpThreads; ++c) above += keys[c] > best;
          if (above == k - 1 && best > floor) sh.floor = best;
          __syncthreads();
          floor = sh.floor > floor ? sh.floor : floor;
          joins = best >= floor;
          __syncthreads();  // everyone has read the floor and the keys
        } else {
          joins = hits();
        }
        if (joins) {
#pragma unroll
          for (int i = 0; i < kLpPer; ++i) {
            const LpKey key = key_of(i);
            if (key != 0 && key >= floor) {
              const int at = atomicAdd(&sh.count[cur], 1);
              if (at < kLpList) sh.list[cur][at] = key;
            }
          }
        }
        if (tid == 0 && floor > sh.floor) sh.floor = floor;
        __syncthreads();
        const int held = min(sh.count[cur], kLpList);
        if (held > k + 32) {
          lp_cut(sh, sh.list[cur], held, k, sh.list[cur ^ 1]);
          __syncthreads();
          if (tid == 0) {
            sh.count[cur ^ 1] = k;
            sh.count[cur] = 0;
          }
          cur ^= 1;
          __syncthreads();
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kLpPer; ++i) v[i] = next[i];
  }

  // ---- the CTA's sums, and its k best in order
  const float wm = warp_max(m);
  if (lane == 0) sh.m[warp] = wm;
  __syncthreads();
  float M = sh.m[0];
#pragma unroll
  for (int i = 1; i < kLpWarps; ++i) M = fmaxf(M, sh.m[i]);
  lp_refer(m, M, s, w, n);
  s = warp_sum(s);
  w = warp_sum(w);
  n = warp_sum(n);
  if (lane == 0) {
    sh.s[warp] = s;
    sh.w[warp] = w;
    sh.n[warp] = n;
  }
  int held = 0;
  if (TOP) {
    held = min(sh.count[cur], kLpList);
    lp_cut(sh, sh.list[cur], held, k, sh.list[cur ^ 1]);
  }
  __syncthreads();
  s = w = n = 0.0f;
#pragma unroll
  for (int i = 0; i < kLpWarps; ++i) {
    s += sh.s[i];
    w += sh.w[i];
    n += sh.n[i];
  }
  const LpKey* ranked = sh.list[cur ^ 1];
  if (splits > 1) {
    if (tid < k) sh.best[tid] = tid < held ? ranked[tid] : 0;
    if (tid == 0) {
      sh.part[0] = M;
      sh.part[1] = s;
      sh.part[2] = w;
      sh.part[3] = n;
    }
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (rank == 0) {
      const bool mine = lane < splits;
      float pm = mine ? lp_remote(&sh.part[0], lane) : -INFINITY;
      s = mine ? lp_remote(&sh.part[1], lane) : 0.0f;
      w = mine ? lp_remote(&sh.part[2], lane) : 0.0f;
      n = mine ? lp_remote(&sh.part[3], lane) : 0.0f;
      M = warp_max(pm);
      lp_refer(pm, M, s, w, n);
      s = warp_sum(s);
      w = warp_sum(w);
      n = warp_sum(n);
      if (TOP) {
        // (0 stands for no key: it is never among the k best of a row of k logits)
        const int all = splits * k;
        LpKey key = 0;
        if (tid < all) key = lp_remote(&sh.best[tid % k], tid / k);
        LpKey* keys = sh.list[cur];
        if (tid < all) keys[tid] = key;
        held = all;
        __syncthreads();
        lp_cut(sh, keys, all, k, sh.list[cur ^ 1]);
        __syncthreads();
      }
    }
  }
  if (rank == 0) {
    const float nan = __uint_as_float(0x7FC00000u);
    s += n - 1.0f;
    const float lse = log1pf(s);
    const bool bad = !(s < INFINITY) || !isfinite(M);
    if (tid == 0) {
      if (bad) flag(a.status, DEV_SOFTMAX);
      if (a.entropy) a.entropy[row] = bad ? nan : lse - w / (1.0f + s);
      if (a.logprob) {
        if (token >= a.vocab) flag(a.status, DEV_TOKEN);
        a.logprob[row] = bad || token >= a.vocab ? nan : token < 0 ? 0.0f : (token_logit - M) - lse;
      }
    }
    if (TOP && tid < k) {
      const LpKey key = ranked[tid];
      const long long o = static_cast<long long>(row) * k + tid;
      a.top_ids[o] = bad ? -1 : lp_index(key);
      a.top_logprobs[o] = bad ? nan : (lp_logit(static_cast<uint32_t>(key >> 32)) - M) - lse;
    }
  }
  if (splits > 1) {  // no CTA leaves while its part may still be read
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  }
}

cudaError_t launch_token_logprobs(LogprobArgs a, int rows, int sms, cudaStream_t st) {
  // CTAs per row: while all are resident at once (four per SM) and each has a
  // segment of its own
  a.splits = 1;
  while (a.splits < kLpCluster && 2LL * rows * a.splits <= 4LL * sms &&
         a.vocab > 4LL * kLpSegment * a.splits)
    a.splits *= 2;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(a.splits), 1, 1};
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  constexpr int kMost = 1 << 27;  // rows of one launch (a grid holds 2^31 - 1 CTAs)
  for (int done = 0; done < rows; done += kMost) {
    const int now = rows - done < kMost ? rows - done : kMost;
    cfg.gridDim = dim3(static_cast<unsigned>(now) * a.splits);
    const cudaError_t e = a.top_k ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<true>, a)
                                  : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<false>, a);
    if (e != cudaSuccess) return e;
    if (rows - done <= kMost) break;
    a.logits += now * a.ld;
    if (a.tokens) a.tokens += now;
    if (a.logprob) a.logprob += now;
    if (a.entropy) a.entropy += now;
    if (a.top_ids) a.top_ids += static_cast<long long>(now) * a.top_k;
    if (a.top_logprobs) a.top_logprobs += static_cast<long long>(now) * a.top_k;
  }
  return cudaSuccess;
}

}  // namespace uocr
