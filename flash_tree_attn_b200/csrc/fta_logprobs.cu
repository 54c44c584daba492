// Log probabilities of given tokens, log-sum-exp, entropy and the likeliest tokens of rows of logits
// (include/fta.h: fta_token_logprobs).
//
// With m the largest logit, s = sum e^(x - m) and t = sum e^(x - m) (x - m):
//   lse = m + log s,  entropy = log s - t / s,  log p(token) = x[token] - lse.
// Every term of t has the same sign, s is 1 and more, and so both terms of the entropy are positive.
//
// What bounds it: the logits are read once; with 16-bit logits an SM gets about 12 elements a clock from
// memory, so there is room for about 10 instructions an element, and 16 exponentials a clock.  So each
// thread keeps sums of its own against its own largest logit so far, with 6 instructions an element (a
// reference that lags behind would save a move a round, and make two large numbers of a peaked row's entropy,
// whose difference then comes out below 0): the exponent is
// x log2(e) - c, c = m log2(e) rounded, one fused multiply-add, and what the rounding of c shifts,
// r = m log2(e) - c, is known exactly and taken out at the end.  Where |m| >= 30000 (logits masked with the
// type's lowest value and nothing else) it is (x - m) log2(e), which cannot overflow.
//
// A row is walked in rounds of 8 chunks of 16 bytes a thread, by one block or, where there are few rows,
// by the blocks of a cluster, which join through distributed shared memory: no workspace and no
// second kernel.
//
// The likeliest: in the first round every warp's q-th largest lane maximum is a bound that at least q of
// the warp's elements reach; the w-th largest of those bounds is reached by q w >= k elements.  Chunks
// whose maximum reaches it (typically less than twice k; later, the k-th largest so far is the bound)
// are listed, their elements shared out over the block and ranked by counting.  Looking at a chunk where
// it was found would hold up its whole warp.  Where more reach the bound than can be listed, the larger
// elements are collected in one more pass and of the equal ones (ties, vocabularies masked with -inf or
// the type's lowest value) the first in order, as many as are wanted; only where the larger ones alone
// are too many is the exact bound found, bit by bit.
#include <cooperative_groups.h>

#include "fta_common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kChunks = 8;        // 16-byte chunks per thread and round
constexpr int kMostBlocks = 8;    // of a cluster, so of a row
// 256 threads a row, 4 blocks an SM: one computes while the others' chunks arrive.  64 threads, or a single
// warp, for many rows of a few thousand logits: such a block's time is its barriers and latencies, and
// more of them fit an SM (26867 rows of 601: 64 threads 37 us, a warp 29).
template <int THREADS> struct Cfg {
  static constexpr int kWarps = THREADS / 32;
  static constexpr int kBlocks = 1024 / THREADS;                   // per SM
  static constexpr int kListedChunks = THREADS == 32 ? 64 : THREADS == 64 ? 128 : 256;
  static constexpr int kListed = 8 * kListedChunks;                // elements ranked by counting
  static constexpr int kPending = THREADS < 256 ? 0 : 64;          // listed chunks that may wait for the next round
  static constexpr int kMostRounds = 32;                           // largest q: a warp's lanes
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// The likeliest go by bits (`ordered`), so what is held against their bound as a float keeps subnormals
// apart too: the compiler's own comparisons take them all for zero (--use_fast_math), and a guard that sees
// equals where the bits differ would let more elements into the list than it holds.
__device__ __forceinline__ bool below(float a, float b) {  // false where either is NaN
  int y;
  asm("{ .reg .pred p; setp.lt.f32 p, %1, %2; selp.s32 %0, 1, 0, p; }" : "=r"(y) : "f"(a), "f"(b));
  return y != 0;
}
__device__ __forceinline__ bool at_most(float a, float b) {
  int y;
  asm("{ .reg .pred p; setp.le.f32 p, %1, %2; selp.s32 %0, 1, 0, p; }" : "=r"(y) : "f"(a), "f"(b));
  return y != 0;
}
__device__ __forceinline__ float max_num(float a, float b) {  // a NaN stays out
  float y;
  asm("max.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// adds 2^d and 2^d d
__device__ __forceinline__ void add_exp(float d, float& s, float& t) {
  const float e = fta_exp2(d);
  s += e;
  t = fmaf(e, d, t);
}

// A 16-byte chunk of logits.  max: NaN if any is.  add: sums over its elements for |m| < 30000; -inf is
// raised to a value whose exponential is still 0, because 0 * -inf is NaN.
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int n = 4;
  static constexpr uint32_t kLowest = 0xff800000u;  // -inf
  static __device__ __forceinline__ float max(const uint4& x) {
    return max_nan(max_nan(__uint_as_float(x.x), __uint_as_float(x.y)), max_nan(__uint_as_float(x.z), __uint_as_float(x.w)));
  }
  static __device__ __forceinline__ void add(const uint4& x, float m2, float& s, float& t) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) add_exp(max_nan(fmaf(__uint_as_float(w[i]), FTA_LOG2E, -m2), -1e30f), s, t);
  }
};
template <> struct Vec<__half> {
  static constexpr int n = 8;
  static constexpr uint32_t kLowest = 0xfc00u;
  static __device__ __forceinline__ __half2 h2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
  static __device__ __forceinline__ float max(const uint4& x) {
    const float2 f = __half22float2(__hmax2_nan(__hmax2_nan(h2(x.x), h2(x.y)), __hmax2_nan(h2(x.z), h2(x.w))));
    return max_nan(f.x, f.y);
  }
  static __device__ __forceinline__ void add(const uint4& x, float m2, float& s, float& t) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(__hmax2_nan(h2(w[i]), h2(0xfbfffbffu)));  // -65504
      add_exp(fmaf(f.x, FTA_LOG2E, -m2), s, t);
      add_exp(fmaf(f.y, FTA_LOG2E, -m2), s, t);
    }
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  static constexpr uint32_t kLowest = 0xff80u;
  static __device__ __forceinline__ __nv_bfloat162 b2(uint32_t x) { return *reinterpret_cast<const __nv_bfloat162*>(&x); }
  static __device__ __forceinline__ uint32_t word(__nv_bfloat162 x) { return *reinterpret_cast<const uint32_t*>(&x); }
  static __device__ __forceinline__ float max(const uint4& x) {
    const uint32_t w = word(__hmax2_nan(__hmax2_nan(b2(x.x), b2(x.y)), __hmax2_nan(b2(x.z), b2(x.w))));
    return max_nan(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ void add(const uint4& x, float m2, float& s, float& t) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t y = word(__hmax2_nan(b2(w[i]), b2(0xfe96fe96u)));  // -1e38: times log2(e) it is finite still
      add_exp(fmaf(__uint_as_float(y << 16), FTA_LOG2E, -m2), s, t);
      add_exp(fmaf(__uint_as_float(y & 0xffff0000u), FTA_LOG2E, -m2), s, t);
    }
  }
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// order of floats as unsigned integers; -0 and +0 alike, NaN on top; 0 is below every float.  The bits are moved
// by hand: of plain casts around operations on the sign bit the compiler makes an absolute value and a
// negation of floats, and those flush subnormals.
__device__ __forceinline__ uint32_t ordered(float x) {
  uint32_t b;
  asm("mov.b32 %0, %1;" : "=r"(b) : "f"(x));
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (b == 0x80000000u) return b;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
  if (k == 0xffffffffu) return NAN;
  const uint32_t b = k & 0x80000000u ? k & 0x7fffffffu : ~k;
  float x;
  asm("mov.b32 %0, %1;" : "=f"(x) : "r"(b));
  return x;
}
// one number that ranks by value, then by lower token
__device__ __forceinline__ unsigned long long rank_key(uint32_t k, int token) {
  return ((unsigned long long)k << 32) | (uint32_t)(0xffffffffu - (uint32_t)token);
}

struct Sums { float m, s, t; };  // s and t (log2 units) relative to m

template <int WARPS> __device__ __forceinline__ int block_sum(int x, int* scratch) {
  x = __reduce_add_sync(0xffffffffu, x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
  __syncthreads();
  int sum = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) sum += scratch[i];
  return sum;
}

// how many of keys[0, n) are larger; the array is zeroed up to a multiple of 8 (the loads of 8 go out
// together: a loop that waits for each of them is most of the time of a small row)
__device__ __forceinline__ int larger(const unsigned long long* keys, int n, unsigned long long own) {
  int before = 0;
  for (int j = 0; j < n; j += 8) {
#pragma unroll
    for (int u = 0; u < 8; u += 2) {
      const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(keys + j + u);
      before += (x.x > own) + (x.y > own);
    }
  }
  return before;
}

__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  if (b.s == 0.f) return a;  // nothing but -inf
  if (a.s == 0.f) return b;
  const float m = fmaxf(a.m, b.m);
  const float da = (a.m - m) * FTA_LOG2E, db = (b.m - m) * FTA_LOG2E, fa = fta_exp2(da), fb = fta_exp2(db);
  return Sums{m, fa * a.s + fb * b.s, (fa == 0.f ? 0.f : fa * (a.t + da * a.s)) + (fb == 0.f ? 0.f : fb * (b.t + db * b.s))};
}

// grid = rows * (blocks of a cluster); block i of a row takes its rounds [i * rounds, (i + 1) * rounds) of
// kThreads * kChunks chunks.  Chunks lie on 16-byte boundaries of memory, whatever the row's start; the few
// elements before the first and behind the last are handed to one lane each.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, Cfg<kThreads>::kBlocks) logprob_kernel(const FtaLogprobParams p, const int blocks, const int rounds) {
  constexpr int VE = Vec<T>::n;
  constexpr int kRound = kThreads * kChunks, kWarps = Cfg<kThreads>::kWarps, kMostRounds = Cfg<kThreads>::kMostRounds;
  constexpr int kListedChunks = Cfg<kThreads>::kListedChunks, kPending = Cfg<kThreads>::kPending;
  // room for what waits from earlier rounds, a whole list, the row's edges, the likeliest so far, and zeros
  constexpr int kRoom = 8 * kPending + Cfg<kThreads>::kListed + 2 * VE;
  __shared__ __align__(16) unsigned long long list[kRoom + FTA_MAX_TOP_K + 8];
  __shared__ unsigned long long best[FTA_MAX_TOP_K];  // the likeliest so far, in order; 0: none
  __shared__ Sums s_sums;
  __shared__ float s_a[kWarps], s_b[kWarps], s_c[kWarps];
  __shared__ int s_i[kWarps];
  __shared__ uint32_t s_key[kWarps];
  __shared__ int s_n, s_larger, s_listed;
  __shared__ int s_where[kListedChunks];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long row = blockIdx.x / blocks;
  const int block = blockIdx.x - (int)row * blocks;
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.l_sr;
  const int head = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int start = min(head ? VE - head : 0, p.vocab);  // the first chunk's first element
  const int total = (p.vocab - start) / VE;               // chunks
  const int k = p.top_k;
  fta_after_previous();
  for (int i = tid; i < k; i += kThreads) best[i] = 0;
  if (tid == 0) s_n = s_larger = s_listed = 0;
  // the first block of a row answers for its tokens; their logits are asked for before all else
  auto logit_of = [&](int i, bool& inside) {
    const long long tok = p.tokens_are_i64 ? reinterpret_cast<const long long*>(p.tokens)[row * p.t_sr + i]
                                           : (long long)reinterpret_cast<const int*>(p.tokens)[row * p.t_sr + i];
    inside = tok >= 0 && tok < p.vocab;
    return inside ? to_float(x[tok]) : -INFINITY;
  };
  // The counts that decide what is appended leave room for it; an index past the room is dropped all the same.
  auto append = [&](uint32_t key, int token) {
    const int to = atomicAdd(&s_listed, 1);
    if (to < kRoom) list[to] = rank_key(key, token);
  };
  bool asked_inside = false;
  const float asked = block == 0 && tid < p.n_tokens ? logit_of(tid, asked_inside) : 0.f;

  // the thread's reference, its rounded log2(e) multiple, what that rounding shifts, and the sums
  float m = -INFINITY, c2 = 0.f, r = 0.f, s = 0.f, t = 0.f;
  bool near = true;
  float bound = -INFINITY;
  int pending = 0;  // listed chunks that wait
  for (int round = 0; round < rounds; ++round) {
    const int base = (block * rounds + round) * kRound;  // first chunk of the round
    const int chunks = min(kRound, total - base);
    if (round > 0) {
      if (chunks <= 0) break;
      if (k > 0) __syncthreads();  // everybody has read the round before's count
    }
    const uint4* at = reinterpret_cast<const uint4*>(x + start + (long long)(base + tid) * VE);
    uint4 raw[kChunks];
    if (chunks == kRound) {
#pragma unroll
      for (int c = 0; c < kChunks; ++c) raw[c] = __ldcs(at + c * kThreads);
    } else {
      const uint32_t low = VE == 8 ? Vec<T>::kLowest * 0x10001u : Vec<T>::kLowest;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        raw[c] = make_uint4(low, low, low, low);
        if (c * kThreads + tid < chunks) raw[c] = __ldcs(at + c * kThreads);
      }
    }
    // lane i of the row's first warp has the i-th element outside the chunks
    int edge = -1;
    float edge_logit = -INFINITY;
    if (block == 0 && round == 0) {
      edge = tid < start ? tid : total * VE + tid;
      if (edge >= p.vocab) edge = -1;
      if (edge >= 0) edge_logit = to_float(x[edge]);
    }

    float top[kChunks], mine = edge_logit;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      top[c] = Vec<T>::max(raw[c]);
      mine = max_nan(mine, top[c]);
    }
    if (mine != mine) {  // so are the row's sums, whatever else the thread has
      s = NAN;
      mine = -INFINITY;
    }

    if (round == 0 && k > 0) {
      // warps whose lanes all hold elements; one that holds part of them will do if k lanes have some
      const int full = max(min(kWarps, chunks / 32), chunks >= k ? 1 : 0);
      const int q = full > 0 ? fta_cdiv(k, full) : kMostRounds + 1;
      uint32_t kth = 0;
      if (q <= kMostRounds && warp < full) {  // the warp's q-th largest lane maximum
        uint32_t key = ordered(mine);
        for (int i = 0; i < q; ++i) {
          kth = __reduce_max_sync(0xffffffffu, key);
          const unsigned who = __ballot_sync(0xffffffffu, key == kth);
          if (lane == __ffs(who) - 1) key = 0;
        }
      }
      if (lane == 0) s_key[warp] = kth;
      __syncthreads();
      if (q <= kMostRounds) {  // the w-th largest of those: the one that w - 1 others come before
        kth = s_key[lane % kWarps];
        int before = 0;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
          const uint32_t o = __shfl_sync(0xffffffffu, kth, i);
          before += o > kth || (o == kth && i < lane % kWarps);
        }
        const unsigned who = __ballot_sync(0xffffffffu, before == fta_cdiv(k, q) - 1);
        bound = unordered(__shfl_sync(0xffffffffu, kth, __ffs(who) - 1));
      }
    }

    if (mine > m) {
      const float to2 = __fmul_rn(mine, FTA_LOG2E);
      near = fabsf(mine) < 30000.f;
      const float r_to = near ? fmaf(mine, FTA_LOG2E, -to2) : 0.f;
      const float shift = (m - mine) * FTA_LOG2E - r + r_to, f = fta_exp2(shift);
      t = f == 0.f ? 0.f : f * (t + shift * s);
      s *= f;
      m = mine; c2 = to2; r = r_to;
    }
    if (mine != -INFINITY) {
      if (near) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          if (c * kThreads >= chunks) break;
          float s1 = 0.f, t1 = 0.f;  // summed per chunk first: the sums' paths stay short
          Vec<T>::add(raw[c], c2, s1, t1);
          s += s1;
          t += t1;
        }
        if (edge >= 0) add_exp(max_nan(fmaf(edge_logit, FTA_LOG2E, -c2), -1e30f), s, t);
      } else {
        for (int c = tid; c < chunks; c += kThreads)
          for (int i = 0; i < VE; ++i) add_exp(max_nan((to_float(x[start + (base + c) * VE + i]) - m) * FTA_LOG2E, -1e30f), s, t);
        if (edge >= 0) add_exp(max_nan((edge_logit - m) * FTA_LOG2E, -1e30f), s, t);
      }
    }
    if (k == 0) continue;

    // list the chunks that reach the bound (NaN does)
    uint32_t reach = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) reach |= below(top[c], bound) ? 0u : 1u << c;
    uint32_t larger_than = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) larger_than |= at_most(top[c], bound) ? 0u : 1u << c;
    while (reach != 0) {
      const int bit = __ffs(reach) - 1, c = bit * kThreads + tid;
      reach &= reach - 1;
      if (c >= chunks) break;
      const int to = atomicAdd(&s_n, 1);
      if (to < kListedChunks) s_where[to] = base + c;
      if ((larger_than >> bit) & 1) atomicAdd(&s_larger, 1);
    }
    if (edge >= 0 && !below(edge_logit, bound)) append(ordered(edge_logit), edge);
    __syncthreads();
    const int reached = s_n;
    if (round > 0 && round + 1 < rounds && base + kRound < total && reached <= kPending) {
      pending = reached;
      continue;
    }
    const bool over = reached > kListedChunks;
    const int listed = over ? pending : reached;  // what earlier rounds listed comes first
    for (int i = tid; i < listed * VE; i += kThreads) {
      const int tok = start + s_where[i / VE] * VE + i % VE;
      const float v = to_float(x[tok]);
      if (!below(v, bound)) append(ordered(v), tok);
    }
    __syncthreads();
    if (over) {
      const int lo = start + base * VE, hi = lo + chunks * VE;
      uint32_t key = ordered(bound);
      if (s_larger > kListedChunks) {
        // the k-th largest value, bit by bit from the top: the largest key that at least k elements reach
        key = 0;
        for (int bit = 31; bit >= 0; --bit) {
          const uint32_t at_least = key | (1u << bit);
          int count = 0;
          for (int i = lo + tid; i < hi; i += kThreads) count += ordered(to_float(x[i])) >= at_least;
          if (block_sum<kWarps>(count, s_i) >= k) key = at_least;
        }
      }
      int larger = 0;
      for (int i = lo + tid; i < hi; i += kThreads) {
        const uint32_t o = ordered(to_float(x[i]));
        if (o > key) {
          append(o, i);
          ++larger;
        }
      }
      int wanted = k - block_sum<kWarps>(larger, s_i);
      for (int first = lo; first < hi && wanted > 0; first += kThreads) {  // in order, until there are enough
        const int i = first + tid;
        const uint32_t o = i < hi ? ordered(to_float(x[i])) : 0u;  // 0: below every key
        const unsigned who = __ballot_sync(0xffffffffu, o == key && i < hi);
        if (lane == 0) s_key[warp] = __popc(who);
        __syncthreads();
        int before = __popc(who & ((1u << lane) - 1)), all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          before += w < warp ? (int)s_key[w] : 0;
          all += s_key[w];
        }
        if (o == key && i < hi && before < wanted) append(o, i);
        wanted -= all;
        __syncthreads();
      }
      __syncthreads();
    }
    int n = min(s_listed, kRoom);
    if (round > 0) {
      for (int i = tid; i < k; i += kThreads) list[n + i] = best[i];
      n += k;
    }
    if (tid < 8) list[n + tid] = 0;
    __syncthreads();
    if (tid == 0) s_n = s_larger = s_listed = 0;
    for (int i = tid; i < n; i += kThreads) {
      const unsigned long long own = list[i];
      const int before = larger(list, n, own);
      if (before < k && own != 0) best[before] = own;
    }
    __syncthreads();
    pending = 0;
    // what comes later has to reach the k-th largest so far; a NaN there stays out of the comparison
    if (best[k - 1] != 0) bound = max_num(bound, unordered((uint32_t)(best[k - 1] >> 32)));
  }

  // the block's sums, against its largest reference
  Sums sums;
  {
    float x = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    if (lane == 0) s_a[warp] = x;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) x = fmaxf(x, s_a[w]);
    const float shift = x == -INFINITY ? 0.f : (m - x) * FTA_LOG2E - r, f = fta_exp2(shift);
    t = f == 0.f ? 0.f : f * (t + shift * s);
    s *= f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      t += __shfl_xor_sync(0xffffffffu, t, o);
    }
    if (lane == 0) { s_b[warp] = s; s_c[warp] = t; }
    __syncthreads();
    sums = Sums{x, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) { sums.s += s_b[w]; sums.t += s_c[w]; }
  }

  // the row's blocks join in the first one
  cg::cluster_group cluster = cg::this_cluster();
  if (blocks > 1) {
    if (tid == 0) s_sums = sums;
    cluster.sync();
    if (block == 0) {
      for (int i = 1; i < blocks; ++i) sums = join(sums, *cluster.map_shared_rank(&s_sums, i));
      for (int i = tid; i < blocks * k; i += kThreads) list[i] = cluster.map_shared_rank(best, i / k)[i % k];
      if (tid < 8) list[blocks * k + tid] = 0;
    }
    cluster.sync();  // the others' shared memory has been read: they may end
    if (block != 0) return;
  } else {
    __syncthreads();
    for (int i = tid; i < k + 8; i += kThreads) list[i] = i < k ? best[i] : 0;
    __syncthreads();
  }
  m = sums.m;
  s = sums.s;
  // the largest logit's term is 1; roundings that take s below it, or t above 0, are put right (NaN stays)
  const float rest = s < 1.f ? 0.f : s - 1.f;
  const float log_s = log1pf(rest);
  if (tid == 0) {
    const float mean = sums.t > 0.f ? 0.f : sums.t / s * FTA_LN2;
    p.lse[row] = s == 0.f ? -INFINITY : m + log_s;
    p.entropy[row] = s == 0.f ? 0.f : log_s - mean;
  }
  // (x - m) - log s: what m and lse have in common is not rounded
  auto log_p = [&](float v) { return s == 0.f || v == -INFINITY ? (s != s ? s : -INFINITY) : (v - m) - log_s; };
  for (int i = tid; i < p.n_tokens; i += kThreads) {
    bool inside = asked_inside;
    const float v = i == tid ? asked : logit_of(i, inside);
    p.logprobs[row * p.n_tokens + i] = inside ? log_p(v) : -INFINITY;
  }
  // Few keys are counted; of many, a key's rank is its place in its own block's list, which is in order, and
  // what a binary search finds before it in the others.
  const bool few = blocks * k <= 64;
  for (int i = tid; i < blocks * k; i += kThreads) {
    const unsigned long long own = list[i];
    if (own == 0) continue;
    int before = few ? larger(list, blocks * k, own) : i % k;
    for (int other = 0; other < blocks && !few; ++other) {
      if (other == i / k) continue;
      int lo = 0, hi = k;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (list[other * k + mid] > own) lo = mid + 1; else hi = mid;
      }
      before += lo;
    }
    if (before < k) {
      p.top_logprobs[row * k + before] = log_p(unordered((uint32_t)(own >> 32)));
      p.top_ids[row * k + before] = (int64_t)(0xffffffffu - (uint32_t)own);
    }
  }
}

template <typename T, int THREADS>
int run_with(const FtaLogprobParams& p, cudaStream_t st) {
  const int chunks = p.vocab / Vec<T>::n, pieces = chunks > 0 ? fta_cdiv(chunks, THREADS * kChunks) : 1;
  // Blocks per row: enough to fill the machine, and no more.  A wave of blocks lasts as long as its
  // rounds, and about one round more for the start and the end of a block, another one for a cluster's join.
  const int slots = kFtaSms * Cfg<THREADS>::kBlocks;
  int blocks = 1, rounds = pieces;
  long long least = 0x7fffffffffffffffLL;
  for (int n = 1; n <= kMostBlocks && n <= pieces; ++n) {
    const int r = fta_cdiv(pieces, n);
    if (fta_cdiv(pieces, r) != n) continue;  // the last block would have nothing
    const long long cost = (((long long)p.rows * n + slots - 1) / slots) * (r + (n > 1 ? 2 : 1));
    if (cost < least) { least = cost; blocks = n; rounds = r; }
  }
  const cudaError_t e = fta_launch_after(logprob_kernel<T, THREADS>, dim3(p.rows * blocks), THREADS, 0, st, blocks, p, blocks, rounds);
  return e == cudaSuccess ? FTA_OK : fta_cuda_fail(e);
}

template <typename T>
int run(const FtaLogprobParams& p, cudaStream_t st) {
  // The first round's bound is loose where k comes near the number of lanes (it is the k-th largest lane
  // maximum at best): a warp's 64 chunks then hold twice or three times k for k up to 16, two warps' 128 for k
  // up to 40; beyond, the lists would overflow, unless they hold all of a row, and the exact bound be searched.
  const int chunks = p.vocab / Vec<T>::n;
  if (p.rows > kFtaSms * 4 && chunks <= 32 * kChunks && p.top_k <= 16) return run_with<T, 32>(p, st);
  if (p.rows > kFtaSms * 4 && chunks <= (p.top_k <= 40 ? 64 * kChunks : Cfg<64>::kListedChunks)) return run_with<T, 64>(p, st);
  return run_with<T, 256>(p, st);
}

}  // namespace

extern "C" int fta_token_logprobs(const FtaLogprobParams* p, void* stream) {
  if (!p || p->rows <= 0 || p->vocab <= 0 || p->top_k < 0 || p->top_k > p->vocab || p->n_tokens < 0) return FTA_E_BADARG;
  if (p->dtype < FTA_DTYPE_F16 || p->dtype > FTA_DTYPE_F32) return FTA_E_BADARG;
  if (!p->logits || !p->entropy || !p->lse || (p->n_tokens > 0 && (!p->tokens || !p->logprobs))) return FTA_E_BADARG;
  if (p->top_k > 0 && (!p->top_logprobs || !p->top_ids)) return FTA_E_BADARG;
  if (reinterpret_cast<uintptr_t>(p->logits) % (p->dtype == FTA_DTYPE_F32 ? 4 : 2) != 0) return FTA_E_BADARG;
  if (p->top_k > FTA_MAX_TOP_K || p->vocab > (1 << 21) || p->rows > (1 << 27)) return FTA_E_UNSUPPORTED;
  cudaStream_t st = (cudaStream_t)stream;
  if (p->dtype == FTA_DTYPE_F16) return run<__half>(*p, st);
  if (p->dtype == FTA_DTYPE_BF16) return run<__nv_bfloat16>(*p, st);
  return run<float>(*p, st);
}
