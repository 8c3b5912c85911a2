// logprobs.cu — log probabilities of given tokens, entropies and the most
// probable alternatives of rows of logits.
//
// Per row x of V logits, M = max x, taken out of the sum once (n elements have
// it), z_i = x_i - M <= 0:
//   S' = sum_{z < 0} e^{z_i} + (n - 1),  log sum e^{z_i} = log1p(S'),
//   log p(t) = z_t - log1p(S'),  H = log1p(S') + (sum e^{z_i} (-z_i)) / (1 + S').
// Leaving the maximum's own 1 out of the sum keeps the log probability of a
// nearly certain token and a nearly zero entropy good to that of their terms: 2.25
// |z| + 4 steps of 2^-24 (z and z log2 e are rounded, exp2 is good to 2 ulp), 2^-16
// where z = -88.  Both terms of H are >= 0, so nothing cancels.
//
// One pass: every warp keeps the maximum of what it has seen and sums that refer
// to it; a new maximum, a rare thing, rescales them.  The alternatives cost the
// loop one 16-bit store: every lane leaves the maximum of each of its turns.
// Behind the loop (or 32 turns) k lanes' best logits give a bound that k elements
// reach, the few turns whose maximum reaches it are read again, their elements
// that do become a short list of candidates, and their rank in it gives the k
// best.  Where the list runs full (thousands of equal logits), or fewer than k
// logits are finite, a second pass bounds every 4096 elements exactly.  A row is
// spread over a cluster of CTAs where the rows are few; the CTAs' sums and lists
// are joined through distributed shared memory.
//
// Bound by the logits' bytes where there are many rows: 1517 rows of 129,280 take
// 118 us without alternatives (6.6 TB/s), 129 us with one, 137 us with twenty.  Few
// rows are bound by latency, most of it of code that runs once: one row takes 5.3 us
// without and 9.7 us with twenty alternatives, 64 rows 9.3 us without (their bytes 5
// us) and 13.1 us with five.  The second pass is slow: where ten logits of a row are
// left and the rest are banned, one row takes 33 us with twenty alternatives, 64 rows 75
// and 1517 rows 988 (with five, which the ten suffice for where a row has one CTA, 136).
#include <cuda_runtime.h>

#include <atomic>

#include "common.cuh"
#include "device_once.h"
#include "kernels.h"

namespace uocr {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpVec = 4;                    // 16-byte vectors per lane and turn
constexpr int kLpPer = 4 * kLpVec;           // elements per lane and turn
constexpr int kLpTurn = 32 * kLpVec;         // vectors per warp and turn: one bulk copy
// Ring slots per warp: two, and four CTAs per SM (1517 rows of 129,280 logits with
// twenty alternatives, as first built, took 152 us; three slots and three CTAs 168, four
// and two 176).
constexpr int kLpStages = 2;
constexpr int kLpCluster = 8;                // most CTAs per row (portable)
constexpr int kLpKept = 32;                  // turns whose maxima are kept
// Terms are summed in FP32, eight of a turn to an accumulator.  Where a warp takes more
// than kLpSerialTurns, they join sums in 64 bits every kLpSerial turns: 512 equal terms
// one after the other are off by 256 steps of 2^-24 at most, but the 262,144 of a flat
// row of 2^30 by 0.4 %.  (In every kernel 0.6 us of 5.2 for one row, 2 % for 1,517.)
constexpr int kLpSerialTurns = 64, kLpSerial = 16;
// Candidates: at most kLpCut stay after a cut, kLogprobMaxTop threads' elements
// join by the exact bound.
constexpr int kLpList = 768;
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
// The upper half of the smallest bf16 >= x, and back.
__device__ __forceinline__ uint16_t lp_up16(float x) {
  const uint32_t u = __float_as_uint(x);
  return static_cast<uint16_t>((u & 0x80000000u ? u : u + 0xFFFFu) >> 16);
}
__device__ __forceinline__ float lp_from16(uint16_t h) {
  return __uint_as_float(static_cast<uint32_t>(h) << 16);
}
// The logit that a candidate reaches: the floor's, but never -inf.
__device__ __forceinline__ float lp_least(LpKey floor) {
  return fmaxf(lp_logit(static_cast<uint32_t>(floor >> 32)), -3.402823466e38f);
}

__device__ __forceinline__ float lp_exp2(float x) {  // 2 ulp
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct LpShared {
  alignas(128) float4 ring[kLpWarps][kLpStages][kLpTurn];
  alignas(16) LpKey list[kLpList + 8];       // zeros up to a multiple of eight when ranked
  uint16_t kept[kLpKept][kLpThreads];        // the lanes' maxima turn by turn (lp_up16)
  LpKey best[kLogprobMaxTop];                // the k best of a cut, in order
  LpKey floor;
  uint64_t full[kLpWarps][kLpStages];
  float m[kLpWarps], s[kLpWarps], w[kLpWarps], n[kLpWarps];
  float part[4];                             // the CTA's {M, S, W, n}
  uint32_t bound[2 * kLogprobMaxTop + kLpWarps];
  int count;                                 // candidates that have joined
  int over;                                  // more than the list holds
  int lost;                                  // a copy has not landed in time
};

// The k best of the list's n, in order, into sh.best; the k-th best, where there
// are k, is the new floor.  All threads; a barrier before and after.
__device__ __noinline__ void lp_rank(LpShared& sh, int n, int k) {
  if (threadIdx.x < 8) sh.list[n + threadIdx.x] = 0;
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < n; i += kLpThreads) {
    const LpKey mine = sh.list[i];
    int rank = 0;
#pragma unroll 1
    for (int c = 0; c < n; c += 8) {
      ulonglong2 o[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] = *reinterpret_cast<const ulonglong2*>(sh.list + c + 2 * u);
#pragma unroll
      for (int u = 0; u < 4; ++u) rank += (o[u].x > mine) + (o[u].y > mine);
    }
    if (rank < k) sh.best[rank] = mine;
    if (rank == k - 1) sh.floor = mine;
  }
}

// The list cut back to its k best (n > k of them).  All threads, between barriers.
__device__ __noinline__ void lp_cut(LpShared& sh, int n, int k) {
  lp_rank(sh, n, k);
  __syncthreads();
  if (threadIdx.x < k) sh.list[threadIdx.x] = sh.best[threadIdx.x];
  if (threadIdx.x == 0) sh.count = k;
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

// Sums S = sum e^{x - m} over all elements but n that equal m, and W = sum
// e^{x - m} (x - m), as they stand to a maximum M >= m.
__device__ __forceinline__ void lp_refer(float m, float M, float& s, float& w, float& n) {
  if (m == M) return;
  const float d = fmaxf(m - M, -1000.0f), f = lp_exp2(d * kLpLog2e), all = s + n;
  w = f * fmaf(d, all, w);
  s = f * all;
  n = 0.0f;
}

// The same for sums in 64 bits, of which none equals the old maximum.
__device__ __noinline__ double2 lp_refer_far(float m, float M, double2 sw) {
  const float d = fmaxf(m - M, -1000.0f);
  const double f = lp_exp2(d * kLpLog2e);
  return make_double2(f * sw.x, f * (sw.y + d * sw.x));
}

__device__ __forceinline__ float lp_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float lp_max_nan(float a, float b) {  // NaN where one is
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// One CTA's elements [e0, e1) of a row: whole 16-byte vectors, and where the row
// does not start or end with one, up to three elements at either end.
struct LpRow {
  const float* x;
  int e0, e1;
  int head, tail;  // elements ahead of the vectors and behind them
  int vecs;        // vectors from element e0 + head

  // Element i of the warp's turn `it` (after the vectors' turns: the ends), as an
  // index of the row.
  __device__ __forceinline__ int index(int it, int turns, int i) const {
    const int lane = threadIdx.x & 31;
    if (it >= turns) return lane < head ? e0 + lane : e1 - tail + lane - head;
    return e0 + head + 4 * (start(it, turns) + (i >> 2) * 32 + lane) + (i & 3);
  }
  // Vectors of each warp's turn: the last turn's are shared out evenly.
  __device__ __forceinline__ int share(int it, int turns) const {
    return it == turns - 1 ? (vecs - it * kLpWarps * kLpTurn + kLpWarps - 1) / kLpWarps : kLpTurn;
  }
  // This warp's first, and how many.
  __device__ __forceinline__ int start(int it, int turns) const {
    return it * kLpWarps * kLpTurn + static_cast<int>(threadIdx.x >> 5) * share(it, turns);
  }
  __device__ __forceinline__ int count(int it, int turns) const {
    return max(0, min(share(it, turns), vecs - start(it, turns)));
  }
};

// Raises the floor to the k-th best of the warps' best lanes: of the r best of each
// warp's 32 orders, r = ceil(2 k / warps), which k elements reach.  A barrier
// before and after.
__device__ __noinline__ void lp_bound(LpShared& sh, uint32_t order, int k) {
  const int r = (2 * k + kLpWarps - 1) / kLpWarps, n = r * kLpWarps;
#pragma unroll 1
  for (int i = 0; i < r; ++i) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, order);
    const unsigned who = __ballot_sync(0xffffffffu, order == top);
    if ((threadIdx.x & 31) == __ffs(who) - 1) {
      order = 0;
      sh.bound[(threadIdx.x >> 5) * r + i] = top;
    }
  }
  __syncthreads();
  if (threadIdx.x < n) {
    const uint32_t mine = sh.bound[threadIdx.x];
    int above = 0, reach = 0;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      above += sh.bound[i] > mine;
      reach += sh.bound[i] >= mine;
    }
    const LpKey floor = static_cast<LpKey>(mine) << 32;  // (equal ones write the same)
    if (above < k && reach >= k && floor > sh.floor) sh.floor = floor;
  }
  __syncthreads();
}

// The elements of this lane's turns [from, to) that reach `least` join the list:
// read again (usually from L2) in the turns whose maximum does.  Code that runs
// once per launch is rolled up: fetching it costs more than running it.
__device__ __noinline__ void lp_join(LpShared& sh, const LpRow& row, int turns, int from, int to,
                                     float least) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t todo = 0;
#pragma unroll 8
  for (int i = 0; i < to - from; ++i)
    if (lp_from16(sh.kept[i][threadIdx.x]) >= least) todo |= 1u << i;
#pragma unroll 1
  for (; todo; todo &= todo - 1) {
    const int it = from + __ffs(todo) - 1;
    uint32_t hits = 0;
    if (it < turns) {
      const float4* vec = reinterpret_cast<const float4*>(row.x + row.e0 + row.head);
      float4 q[kLpVec];
#pragma unroll
      for (int r = 0; r < kLpVec; ++r) {
        q[r] = r * 32 + lane < row.count(it, turns)
                   ? vec[row.start(it, turns) + r * 32 + lane]
                   : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      }
#pragma unroll
      for (int r = 0; r < kLpVec; ++r)
        hits |= ((q[r].x >= least ? 1u : 0u) | (q[r].y >= least ? 2u : 0u) | (q[r].z >= least ? 4u : 0u) |
                 (q[r].w >= least ? 8u : 0u)) << (4 * r);
    } else if (warp == 0 && lane < row.head + row.tail) {
      hits = 1;
    }
#pragma unroll 1
    for (; hits; hits &= hits - 1) {
      const int e = row.index(it, turns, __ffs(hits) - 1);
      const int at = atomicAdd(&sh.count, 1);
      if (at < kLpList) sh.list[at] = lp_key(row.x[e], e);
    }
  }
}

// The candidates of the CTA's elements picked again, whatever the logits are:
// every 4096 elements bounded by the k-th best of the threads' best keys, which
// only k threads reach.  The list ends with all of the k best in it.
__device__ __noinline__ void lp_pick_exactly(LpShared& sh, const LpRow& row, int k) {
  const int tid = threadIdx.x;
  LpKey* keys = reinterpret_cast<LpKey*>(sh.ring);  // (every copy has landed and been read)
  if (tid == 0) sh.count = 0;
#pragma unroll 1
  for (int first = row.e0; first < row.e1; first += kLpThreads * kLpPer) {
    LpKey best = 0;
#pragma unroll 4
    for (int i = 0; i < kLpPer; ++i) {
      const int e = first + i * kLpThreads + tid;
      const float v = e < row.e1 ? row.x[e] : 0.0f;
      const LpKey key = e < row.e1 && !isnan(v) ? lp_key(v, e) : 0;
      best = key > best ? key : best;
    }
    __syncthreads();
    keys[tid] = best;
    __syncthreads();
    int above = 0;
#pragma unroll 4
    for (int c = 0; c < kLpThreads; c += 2) {
      const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(keys + c);
      above += (o.x > best) + (o.y > best);
    }
    if (above == k - 1 && best > sh.floor) sh.floor = best;  // (one thread, the only reader)
    __syncthreads();
    const LpKey floor = sh.floor;
    if (best >= floor) {
#pragma unroll 1
      for (int i = 0; i < kLpPer; ++i) {
        const int e = first + i * kLpThreads + tid;
        if (e >= row.e1) break;
        const float v = row.x[e];
        const LpKey key = isnan(v) ? 0 : lp_key(v, e);
        if (key != 0 && key >= floor) sh.list[atomicAdd(&sh.count, 1)] = key;
      }
    }
    __syncthreads();
    const int held = sh.count;
    if (held > kLpCut) lp_cut(sh, held, k);  // room for the next 4096's
    __syncthreads();
  }
  __syncthreads();
}

// The copies of the warp's turns from `it` on have not landed in time (a safety net:
// flagged): those in flight, before turn `end`, are waited for again, so that none
// lands behind the CTA's end.
__device__ __noinline__ void lp_give_up(LpShared& sh, int it, int end, unsigned* status, long long cycles) {
#pragma unroll 1
  for (int i = it; i < it + kLpStages && i < end; ++i)
    mbar_wait_try(&sh.full[threadIdx.x >> 5][i % kLpStages], i / kLpStages & 1, status, cycles);
  sh.lost = 1;  // (read behind barriers)
}

// TOP: alternatives; LONG: rows of many turns.
template <bool TOP, bool LONG>
__global__ void __launch_bounds__(kLpThreads, 4) token_logprobs_kernel(const LogprobArgs a) {
  extern __shared__ __align__(128) unsigned char lp_raw[];
  LpShared& sh = *reinterpret_cast<LpShared*>(lp_raw);
  pdl_launch_dependents();  // launched as a programmatic dependent (launch_dependent):
  pdl_wait_prior_grids();   // nothing is touched before the previous kernel completes
  const int splits = a.splits, rank = blockIdx.x % splits, row = blockIdx.x / splits;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, k = a.top_k;
  LpRow part;
  part.x = a.logits + row * a.ld;
  {
    const int skip = static_cast<int>((reinterpret_cast<uintptr_t>(part.x) >> 2) & 3);
    const int head = skip ? min(4 - skip, a.vocab) : 0;
    const int vecs = (a.vocab - head) >> 2;  // of the row
    const int first = static_cast<int>(static_cast<long long>(vecs) * rank / splits);
    const int last = static_cast<int>(static_cast<long long>(vecs) * (rank + 1) / splits);
    part.vecs = last - first;
    part.head = rank == 0 ? head : 0;
    part.tail = rank == splits - 1 ? a.vocab - head - 4 * vecs : 0;
    part.e0 = rank == 0 ? 0 : head + 4 * first;
    part.e1 = rank == splits - 1 ? a.vocab : head + 4 * last;
  }
  // turns of every warp: a bulk copy of up to kLpTurn vectors each; one more for
  // the elements at the ends
  const int turns = (part.vecs + kLpWarps * kLpTurn - 1) / (kLpWarps * kLpTurn);
  const int all_turns = turns + (part.head + part.tail > 0);
  auto fetch = [&](int it, int slot) {
    const int n = part.count(it, turns);
    if (n == 0) return;
    mbar_arrive_expect_tx(&sh.full[warp][slot], n * 16);
    bulk_g2s(sh.ring[warp][slot],
             part.x + part.e0 + part.head + 4LL * part.start(it, turns), n * 16,
             &sh.full[warp][slot]);
  };
  if (lane == 0) {
    for (int i = 0; i < kLpStages; ++i) mbar_init(&sh.full[warp][i], 1 + a.wait.extra);
    fence_mbar_init();
    for (int i = 0; i < kLpStages && i < turns; ++i) fetch(i, i);
  }
  long long token = -1;
  float token_logit = 0.0f;
  if (a.tokens && rank == 0 && tid == 0) {
    token = a.tokens[row];
    if (token >= 0 && token < a.vocab) token_logit = part.x[token];
  }
  if (tid == 0) {
    sh.count = 0;
    sh.over = 0;
    sh.lost = 0;
    sh.floor = 0;
  }
  __syncthreads();
  // The warp's maximum so far, and sums that refer to it and leave one instance of
  // it out, in the lane whose n is 1.
  float m = -INFINITY, n = 0.0f;
  double2 far = make_double2(0.0, 0.0);  // both, of the turns that are no longer in s2, w2
  float2 s2 = make_float2(0.0f, 0.0f), w2 = make_float2(0.0f, 0.0f);
  float best = -INFINITY;  // of this lane, since turn `from`
  int from = 0;
  int stop = turns;  // where a wait gives up: its turn; no more copies are waited for or started
  // the candidates of turns [from, to)
  auto gather = [&](int to) {
    lp_bound(sh, lp_order(best), k);
    lp_join(sh, part, turns, from, to, lp_least(sh.floor));
    __syncthreads();
  };
#pragma unroll 1
  for (int it = 0, slot = 0, phase = 0; it < all_turns; ++it) {
    float v[kLpPer];
    const int here = it < stop ? part.count(it, turns) : 0;
    if (here == kLpTurn) {
      if (!mbar_wait_try(&sh.full[warp][slot], phase, a.status, a.wait.cycles)) stop = it;
#pragma unroll
      for (int r = 0; r < kLpVec; ++r) {
        const float4 q = sh.ring[warp][slot][r * 32 + lane];
        v[4 * r] = q.x;
        v[4 * r + 1] = q.y;
        v[4 * r + 2] = q.z;
        v[4 * r + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kLpPer; ++i) v[i] = -INFINITY;
      if (here > 0) {
        if (!mbar_wait_try(&sh.full[warp][slot], phase, a.status, a.wait.cycles)) stop = it;
#pragma unroll
        for (int r = 0; r < kLpVec; ++r)
          if (r * 32 + lane < here) {
            const float4 q = sh.ring[warp][slot][r * 32 + lane];
            v[4 * r] = q.x;
            v[4 * r + 1] = q.y;
            v[4 * r + 2] = q.z;
            v[4 * r + 3] = q.w;
          }
      } else if (it >= turns && warp == 0 && lane < part.head + part.tail) {
        v[0] = part.x[part.index(it, turns, 0)];
      }
    }
    float mx = v[0];
#pragma unroll
    for (int i = 1; i + 1 < kLpPer; i += 2) mx = lp_max3(mx, v[i], v[i + 1]);
    mx = fmaxf(mx, v[kLpPer - 1]);
    if (TOP) {
      best = fmaxf(best, mx);
      sh.kept[it - from][tid] = lp_up16(mx);
    }
    __syncwarp();  // every lane has read the slot
    if (lane == 0 && it + kLpStages < stop) fetch(it + kLpStages, slot);
    if (++slot == kLpStages) {
      slot = 0;
      phase ^= 1;
    }
    if (__any_sync(0xffffffffu, mx > m)) {
      // a new maximum of the warp: the old one joins its lane's sums, one instance
      // of the new one leaves
      const float top = warp_max(mx > m ? mx : m);
      float s = s2.x + s2.y, w = w2.x + w2.y;
      lp_refer(m, top, s, w, n);
      s2 = make_float2(s, 0.0f);
      w2 = make_float2(w, 0.0f);
      if (LONG && it >= kLpSerial) far = lp_refer_far(m, top, far);
      m = top;
      const unsigned who = __ballot_sync(0xffffffffu, mx == m);
      if (lane == __ffs(who) - 1) {
        n = 1.0f;
        bool left = false;
#pragma unroll
        for (int i = 0; i < kLpPer; ++i) {
          const bool it_is = !left && v[i] == mx;
          left |= it_is;
          v[i] = it_is ? -INFINITY : v[i];
        }
      }
    }
    const float ref = m == -INFINITY ? 0.0f : -m;
#pragma unroll
    for (int i = 0; i < kLpPer; i += 2) {
      // z from -1000 up (e^z is 0 there, and e^z z is 0 too, not NaN); NaN stays
      float2 z = f2_add(make_float2(v[i], v[i + 1]), make_float2(ref, ref));
      z = make_float2(lp_max_nan(z.x, -1000.0f), lp_max_nan(z.y, -1000.0f));
      const float2 y = f2_mul(z, make_float2(kLpLog2e, kLpLog2e));
      const float2 e = make_float2(lp_exp2(y.x), lp_exp2(y.y));
      s2 = f2_add(s2, e);
      w2 = f2_fma(e, z, w2);
    }
    if (LONG && it % kLpSerial == kLpSerial - 1) {
      far.x += s2.x + s2.y;
      far.y += w2.x + w2.y;
      s2 = w2 = make_float2(0.0f, 0.0f);
    }
    if (TOP && it + 1 - from == kLpKept && it + 1 < all_turns) {
      gather(it + 1);
      const int held = sh.count;  // (written next behind a barrier)
      if (held > kLpList) {
        if (tid == 0) sh.over = 1;
      } else if (held > kLpCut) {
        lp_cut(sh, held, k);
      }
      __syncthreads();
      if (tid == 0 && held > kLpList) sh.count = 0;  // (the second pass will pick)
      from = it + 1;
      best = -INFINITY;
    }
  }
  float s = s2.x + s2.y, w = w2.x + w2.y;
  if (LONG) {
    s = static_cast<float>(far.x + s);
    w = static_cast<float>(far.y + w);
  }
  if (stop < turns) {
    lp_give_up(sh, stop, part.count(turns - 1, turns) ? turns : turns - 1, a.status, a.wait.cycles);
    s = __uint_as_float(0x7FC00000u);  // (the row is NaN)
  }
  if (TOP && all_turns) gather(all_turns);

  // ---- the CTA's sums, and its k best in order
  if (lane == 0) sh.m[warp] = m;
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
  if (TOP) {  // (every join lies behind the barrier above)
    const bool gone = sh.lost;  // (the row is NaN, and the ring may still be written)
    held = gone ? 0 : sh.count;
    // the list has run full, or k logits that are not -inf have not been found
    if (!gone && (sh.over || held > kLpList || (held < k && held < part.e1 - part.e0))) {
      __syncthreads();
      lp_pick_exactly(sh, part, k);
      held = sh.count;
    }
    lp_rank(sh, held, k);
  }
  __syncthreads();
  s = w = n = 0.0f;
#pragma unroll
  for (int i = 0; i < kLpWarps; ++i) {
    s += sh.s[i];
    w += sh.w[i];
    n += sh.n[i];
  }
  if (splits > 1) {
    if (tid >= held && tid < k) sh.best[tid] = 0;
    if (tid == 0) sh.count = 0;
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
      const float pm = mine ? lp_remote(&sh.part[0], lane) : -INFINITY;
      s = mine ? lp_remote(&sh.part[1], lane) : 0.0f;
      w = mine ? lp_remote(&sh.part[2], lane) : 0.0f;
      n = mine ? lp_remote(&sh.part[3], lane) : 0.0f;
      // the parts' k best (0 behind their ends: never among those of a row of k
      // logits); k of them reach the least of the parts' r-th best, r = ceil(k / splits)
      LpKey key = 0, least = ~0ull;
      if (TOP && tid < splits * k) key = lp_remote(&sh.best[tid % k], tid / k);
      if (TOP && mine) least = lp_remote(&sh.best[(k + splits - 1) / splits - 1], lane);
      M = pm;
#pragma unroll
      for (int o = 1; o < kLpCluster; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
      M = __shfl_sync(0xffffffffu, M, 0);
      lp_refer(pm, M, s, w, n);
#pragma unroll
      for (int o = 1; o < kLpCluster; o <<= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        w += __shfl_xor_sync(0xffffffffu, w, o);
        n += __shfl_xor_sync(0xffffffffu, n, o);
      }
      s = __shfl_sync(0xffffffffu, s, 0);
      w = __shfl_sync(0xffffffffu, w, 0);
      n = __shfl_sync(0xffffffffu, n, 0);
      if (TOP) {
#pragma unroll
        for (int o = 1; o < kLpCluster; o <<= 1) {
          const LpKey other = __shfl_xor_sync(0xffffffffu, least, o);
          least = other < least ? other : least;
        }
        least = __shfl_sync(0xffffffffu, least, 0);
        if (key != 0 && key >= least) sh.list[atomicAdd(&sh.count, 1)] = key;
        __syncthreads();
        lp_rank(sh, sh.count, k);
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
      const LpKey key = sh.best[tid];
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

// Clusters of `splits` CTAs that fit the device at once with `per` CTAs on an SM,
// asked once per device (0 where the answer is an error).
static int lp_clusters(int splits, int per, cudaLaunchConfig_t cfg) {
  static std::atomic<int> known[64][9][5];  // answer + 1
  int dev = 0;
  cudaGetDevice(&dev);
  std::atomic<int>* at = dev >= 0 && dev < 64 ? &known[dev][splits][per] : nullptr;
  if (at && at->load(std::memory_order_relaxed)) return at->load(std::memory_order_relaxed) - 1;
  int n = 0;
  cfg.gridDim = dim3(splits);
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, token_logprobs_kernel<true, false>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  if (at) at->store(n + 1, std::memory_order_relaxed);
  return n;
}

cudaError_t launch_token_logprobs(LogprobArgs a, int rows, int sms, cudaStream_t st) {
  constexpr size_t smem = sizeof(LpShared);
  constexpr int kLpSmemSm = 228 * 1024;  // of an SM, 1 KB of it the system's per CTA
  static_assert(4 * (smem + 1024) <= kLpSmemSm, "four CTAs per SM");
  static PerDeviceOnce configured;
  configured.run([] {
    for (auto kernel : {token_logprobs_kernel<true, false>, token_logprobs_kernel<true, true>,
                        token_logprobs_kernel<false, false>, token_logprobs_kernel<false, true>})
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kLpSmemSm / 2 - 1024);
  });
  // CTAs per row: while three per SM hold them all and each has a full ring (64
  // rows of 129,280 logits with five alternatives: 15.2 us by 4, 16.4 by 8, 19.3 by
  // 2; 40 rows 13.4 by 8, 14.4 by 4; 300 rows 40.5 by 1, 44.1 by 2)
  a.splits = 1;
  while (a.splits < kLpCluster && 2LL * rows * a.splits <= 3LL * sms &&
         a.vocab > 4LL * kLpTurn * kLpWarps * a.splits)
    a.splits *= 2;
  const bool far = a.vocab > static_cast<long long>(kLpSerialTurns) * kLpTurn * 4 * kLpWarps * a.splits;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(a.splits), 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  // Clusters are packed onto as few SMs as hold them: where two or three CTAs per
  // SM hold all of them, a CTA asks for more shared memory than it uses, so that
  // no more share one (150 rows of 129,280 logits: 34.4 -> 18.2 us).
  cfg.dynamicSmemBytes = smem;
  for (int per = 2; per < 4; ++per) {
    cudaLaunchConfig_t wide = cfg;
    wide.dynamicSmemBytes = kLpSmemSm / per - 1024;
    if (lp_clusters(a.splits, per, wide) >= rows) {
      cfg.dynamicSmemBytes = wide.dynamicSmemBytes;
      break;
    }
  }
  constexpr int kMost = 1 << 27;  // rows of one launch (a grid holds 2^31 - 1 CTAs)
  for (int done = 0; done < rows; done += kMost) {
    const int now = rows - done < kMost ? rows - done : kMost;
    cfg.gridDim = dim3(static_cast<unsigned>(now) * a.splits);
    auto kernel = a.top_k ? far ? token_logprobs_kernel<true, true> : token_logprobs_kernel<true, false>
                  : far   ? token_logprobs_kernel<false, true>
                          : token_logprobs_kernel<false, false>;
    cfg.numAttrs = 2;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e != cudaSuccess) {  // without the early start
      cudaGetLastError();
      cfg.numAttrs = 1;
      e = cudaLaunchKernelEx(&cfg, kernel, a);
    }
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
