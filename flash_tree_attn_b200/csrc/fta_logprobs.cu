// Log probabilities of given tokens, log-sum-exp, entropy and the likeliest tokens of rows of logits
// (include/fta.h: fta_token_logprobs).
//
// With m the largest logit, s = sum e^(x - m) and t = sum e^(x - m) (x - m):
//   lse = m + log s,  entropy = log s - t / s,  log p(token) = x[token] - lse.
// Every term of t has the same sign, so the entropy loses nothing but in the last difference.
//
// Where |m| < 30000 the exponents are x log2(e) - m2 with m2 = m log2(e) rounded, one fused multiply-add
// an element; what the rounding of m2 shifts, r = m log2(e) - m2, is known exactly and taken out of the
// piece's sums.  Elsewhere (logits masked with the type's lowest value and nothing else) they are
// (x - m) log2(e), which cannot overflow.
//
// What bounds it: the logits are read once; with 16-bit logits an SM gets about 12 elements a clock from
// memory, so there is room for about 10 instructions an element, and 16 exponentials a clock.  A row is
// cut into pieces that a block holds in registers (8 chunks of 16 bytes a thread), so the maximum (packed,
// per chunk), the sums (6 instructions an element) and the search for the likeliest need no second
// read, and a few long rows spread over the machine.  A second kernel joins the pieces.
//
// The likeliest of a piece: every warp's q-th largest of its lanes' maxima is a bound that at least q
// of the warp's elements reach; the least of those bounds over W warps is reached by q W >= k elements.
// Only chunks whose maximum reaches it are looked at again (typically two or three times k elements
// do), and what is found is ranked by counting.  Where too many do (ties, masked vocabularies) the exact
// bound is found bit by bit instead.
#include "fta_common.cuh"

namespace {

constexpr int kThreads = 256;     // 4 blocks an SM: one computes while the others' chunks arrive
constexpr int kWarps = kThreads / 32;
constexpr int kChunks = 8;        // 16-byte chunks per thread
constexpr int kListed = 1024;     // elements ranked by counting
constexpr int kMostRounds = 16;   // largest q; below 4 full warps a piece has fewer than kListed elements
constexpr int kJoin = 128;

__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// adds 2^d and 2^d d
__device__ __forceinline__ void add_exp(float d, float& s, float& t) {
  const float e = fta_exp2(d);
  s += e;
  t = fmaf(e, d, t);
}

// A 16-byte chunk of logits.  max: NaN if any is.  add: sums over its elements for |m| < 30000; -inf is
// raised to a value whose exponential is still 0, because 0 * -inf is NaN.  get: element i.
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int n = 4;
  static constexpr uint32_t kLowest = 0xff800000u;  // -inf
  static __device__ __forceinline__ uint32_t bits(const float* x) { return __float_as_uint(*x); }
  static __device__ __forceinline__ float max(const uint4& x) {
    return max_nan(max_nan(__uint_as_float(x.x), __uint_as_float(x.y)), max_nan(__uint_as_float(x.z), __uint_as_float(x.w)));
  }
  static __device__ __forceinline__ void add(const uint4& x, float m2, float& s, float& t) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) add_exp(max_nan(fmaf(__uint_as_float(w[i]), FTA_LOG2E, -m2), -1e30f), s, t);
  }
  static __device__ __forceinline__ float get(uint32_t w, int) { return __uint_as_float(w); }
};
template <> struct Vec<__half> {
  static constexpr int n = 8;
  static constexpr uint32_t kLowest = 0xfc00u;
  static __device__ __forceinline__ uint32_t bits(const __half* x) { return __half_as_ushort(*x); }
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
  static __device__ __forceinline__ float get(uint32_t w, int i) { return __half2float(__ushort_as_half((unsigned short)(i ? w >> 16 : w & 0xffffu))); }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  static constexpr uint32_t kLowest = 0xff80u;
  static __device__ __forceinline__ uint32_t bits(const __nv_bfloat16* x) { return __bfloat16_as_ushort(*x); }
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
  static __device__ __forceinline__ float get(uint32_t w, int i) { return __uint_as_float(i ? w & 0xffff0000u : w << 16); }
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// order of floats as unsigned integers; -0 and +0 alike, NaN on top; 0 is below every float
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (b == 0x80000000u) return b;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
  if (k == 0xffffffffu) return NAN;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// one number that ranks by value, then by lower token
__device__ __forceinline__ unsigned long long rank_key(uint32_t k, int token) {
  return ((unsigned long long)k << 32) | (uint32_t)(0xffffffffu - (uint32_t)token);
}

struct Piece { float m, s, t, unused; };

template <int N> __device__ __forceinline__ int block_sum(int x, int* scratch) {
  x = __reduce_add_sync(0xffffffffu, x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = x;
  __syncthreads();
  int sum = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) sum += scratch[i];
  return sum;
}

// grid = rows * pieces.  Chunks lie on 16-byte boundaries of memory, whatever the row's start: element
// e of the row is element e + head of the chunks.
template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_piece_kernel(const FtaLogprobParams p, const int pieces) {
  constexpr int VE = Vec<T>::n;
  static_assert(kThreads * kChunks * VE <= 1 << 15, "the search over a piece's tokens takes 16 steps");
  __shared__ unsigned long long list[kListed];
  __shared__ float s_a[kWarps], s_b[kWarps], s_c[kWarps];
  __shared__ int s_i[kWarps];
  __shared__ int s_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long row = blockIdx.x / pieces;
  const int piece = blockIdx.x - (int)row * pieces;
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.l_sr;
  const int head = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int base = piece * (kThreads * kChunks);  // first chunk of the piece
  const int k = p.top_k;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join's blocks wait for this grid's end

  uint4 raw[kChunks];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int e0 = (base + c * kThreads + tid) * VE - head;
    if (e0 >= 0 && e0 + VE <= p.vocab) {
      raw[c] = __ldcs(reinterpret_cast<const uint4*>(x + e0));
    } else {  // the row's ends
      uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const uint32_t v = e0 + i >= 0 && e0 + i < p.vocab ? Vec<T>::bits(x + e0 + i) : Vec<T>::kLowest;
        w[i * 4 / VE] |= v << (VE == 8 ? 16 * (i & 1) : 0);
      }
      raw[c] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  float top[kChunks], mine = -INFINITY;
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    top[c] = Vec<T>::max(raw[c]);
    mine = fmaxf(mine, top[c]);
  }
  float m = mine;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));

  // the warp's bound: its q-th largest lane maximum
  const int chunks = min(kThreads * kChunks, fta_cdiv(p.vocab + head, VE) - base);  // of this piece
  const int full = min(kWarps, (chunks - (head > 0 && piece == 0 ? 1 : 0)) / 32);    // warps whose lanes all hold elements
  float bound = -INFINITY;
  if (k > 0 && full > 0 && fta_cdiv(k, full) <= kMostRounds) {
    const int q = fta_cdiv(k, full);
    uint32_t key = ordered(mine);
    if (warp < full) {
      uint32_t kth = 0;
      for (int i = 0; i < q; ++i) {
        kth = __reduce_max_sync(0xffffffffu, key);
        const unsigned who = __ballot_sync(0xffffffffu, key == kth);
        if (lane == __ffs(who) - 1) key = 0;
      }
      bound = unordered(kth);
    } else {
      bound = INFINITY;
    }
  }
  if (lane == 0) { s_a[warp] = m; s_b[warp] = bound; }
  if (tid == 0) s_n = 0;
  __syncthreads();
  m = -INFINITY;
  bound = INFINITY;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) { m = fmaxf(m, s_a[w]); bound = fminf(bound, s_b[w]); }

  const bool near = fabsf(m) < 30000.f;
  const float m2 = __fmul_rn(m, FTA_LOG2E), safe = m == -INFINITY ? 0.f : m;
  float s = 0.f, t = 0.f;
  if (near) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
      if (c * kThreads < chunks) Vec<T>::add(raw[c], m2, s, t);
  } else {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
      for (int i = 0; i < VE; ++i) add_exp(max_nan((Vec<T>::get(w[i * 4 / VE], i & 1) - safe) * FTA_LOG2E, -1e30f), s, t);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
  }
  __syncthreads();
  if (lane == 0) { s_b[warp] = s; s_c[warp] = t; }
  __syncthreads();
  uint8_t* ws = reinterpret_cast<uint8_t*>(p.workspace);
  if (tid == 0) {
    s = t = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) { s += s_b[w]; t += s_c[w]; }
    if (near) {  // 2^(x log2(e) - m2) = e^(x - m) 2^r
      const float r = fmaf(m, FTA_LOG2E, -m2), f = fta_exp2(-r);
      t = f * (t - r * s);
      s *= f;
    }
    reinterpret_cast<Piece*>(ws)[row * pieces + piece] = Piece{m, s, t, 0.f};
  }
  if (k == 0) return;

  // list what reaches the bound (NaN does): the few chunks that do are read again, from the cache
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    if (top[c] < bound || c * kThreads >= chunks) continue;
    const int tok0 = (base + c * kThreads + tid) * VE - head;
    for (int i = max(0, -tok0); i < VE && tok0 + i < p.vocab; ++i) {
      const float v = to_float(x[tok0 + i]);
      if (v < bound) continue;
      const int at = atomicAdd(&s_n, 1);
      if (at < kListed) list[at] = rank_key(ordered(v), tok0 + i);
    }
  }
  __syncthreads();
  int n = s_n;
  if (n > kListed) {
    const int lo = max(0, base * VE - head), hi = min(p.vocab, (base + kThreads * kChunks) * VE - head);
    // The k-th largest value, bit by bit from the top: the largest key that at least k elements reach.
    uint32_t key = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t at_least = key | (1u << bit);
      int count = 0;
      for (int i = lo + tid; i < hi; i += kThreads) count += ordered(to_float(x[i])) >= at_least;
      if (block_sum<kWarps>(count, s_i) >= k) key = at_least;
    }
    // Of the elements equal to it the lowest tokens are wanted: those below the least `end` that makes k.
    int end = lo;
    for (int step = 1 << 15; step > 0; step >>= 1) {  // a piece holds at most 2^15 elements
      int count = 0;
      for (int i = lo + tid; i < hi; i += kThreads) {
        const uint32_t o = ordered(to_float(x[i]));
        count += o > key || (o == key && i < end + step);
      }
      if (block_sum<kWarps>(count, s_i) < k) end += step;
    }
    if (tid == 0) s_n = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += kThreads) {
      const uint32_t o = ordered(to_float(x[i]));
      if (o > key || (o == key && i <= end)) list[atomicAdd(&s_n, 1)] = rank_key(o, i);
    }
    __syncthreads();
    n = s_n;
  }
  unsigned long long* out = reinterpret_cast<unsigned long long*>(ws + (long long)p.rows * pieces * sizeof(Piece)) + (row * pieces + piece) * k;
  for (int i = tid; i < n; i += kThreads) {
    const unsigned long long own = list[i];
    int before = 0;
    for (int j = 0; j < n; ++j) before += list[j] > own;
    if (before < k) out[before] = own;
  }
  for (int i = n + tid; i < k; i += kThreads) out[i] = 0;  // a short last piece
}

// grid = rows: joins a row's pieces.
template <typename T>
__global__ void __launch_bounds__(kJoin) logprob_join_kernel(const FtaLogprobParams p, const int pieces) {
  extern __shared__ unsigned long long keys[];
  const long long row = blockIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint8_t* ws = reinterpret_cast<const uint8_t*>(p.workspace);
  const Piece* part = reinterpret_cast<const Piece*>(ws) + row * pieces;
  float m = -INFINITY, s = 0.f, t = 0.f;
  for (int i = 0; i < pieces; ++i) m = fmaxf(m, part[i].m);
  for (int i = 0; i < pieces; ++i) {
    const Piece q = part[i];
    if (q.s == 0.f) continue;  // nothing but -inf
    const float shift = (q.m - m) * FTA_LOG2E;
    const float f = fta_exp2(shift);
    s += f * q.s;
    t += f == 0.f ? 0.f : f * (q.t + shift * q.s);
  }
  const float log2_s = fta_log2(s);
  const float log_s = log2_s * FTA_LN2;
  const float lse = s == 0.f ? -INFINITY : m + log_s;
  if (threadIdx.x == 0) {
    p.lse[row] = lse;
    p.entropy[row] = s == 0.f ? 0.f : (log2_s - t / s) * FTA_LN2;
  }
  // (x - m) - log s: what m and lse have in common is not rounded
  auto log_p = [&](float v) { return s == 0.f || v == -INFINITY ? (s != s ? s : -INFINITY) : (v - m) - log_s; };
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.l_sr;
  for (int i = threadIdx.x; i < p.n_tokens; i += kJoin) {
    const long long tok = p.tokens_are_i64 ? reinterpret_cast<const long long*>(p.tokens)[row * p.t_sr + i]
                                           : (long long)reinterpret_cast<const int*>(p.tokens)[row * p.t_sr + i];
    float lp = -INFINITY;
    if (tok >= 0 && tok < p.vocab) lp = log_p(to_float(x[tok]));
    p.logprobs[row * p.n_tokens + i] = lp;
  }
  if (p.top_k == 0) return;
  const int n = pieces * p.top_k;
  const unsigned long long* in = reinterpret_cast<const unsigned long long*>(ws + (long long)p.rows * pieces * sizeof(Piece)) + row * n;
  for (int i = threadIdx.x; i < n; i += kJoin) keys[i] = in[i];
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kJoin) {
    const unsigned long long own = keys[i];
    if (own == 0) continue;
    int before = 0;
    for (int j = 0; j < n; ++j) before += keys[j] > own;
    if (before < p.top_k) {
      p.top_logprobs[row * p.top_k + before] = log_p(unordered((uint32_t)(own >> 32)));
      p.top_ids[row * p.top_k + before] = (int64_t)(0xffffffffu - (uint32_t)own);
    }
  }
}

int pieces_of(const FtaLogprobParams& p) {
  const int ve = p.dtype == FTA_DTYPE_F32 ? 4 : 8;
  // a row's start may push its elements up to ve - 1 places into the chunks
  return fta_cdiv(p.vocab + ve - 1, kThreads * kChunks * ve);
}

int check_sizes(const FtaLogprobParams* p) {
  if (!p || p->rows <= 0 || p->vocab <= 0 || p->top_k < 0 || p->top_k > p->vocab || p->n_tokens < 0) return FTA_E_BADARG;
  if (p->dtype < FTA_DTYPE_F16 || p->dtype > FTA_DTYPE_F32) return FTA_E_BADARG;
  if (p->top_k > FTA_MAX_TOP_K || p->vocab > (1 << 19)) return FTA_E_UNSUPPORTED;
  if ((long long)p->rows * pieces_of(*p) > 0x7fffffffLL) return FTA_E_UNSUPPORTED;
  return FTA_OK;
}

int64_t ws_bytes(const FtaLogprobParams& p) { return (int64_t)p.rows * pieces_of(p) * (sizeof(Piece) + 8 * p.top_k); }

template <typename T>
int run(const FtaLogprobParams& p, cudaStream_t st) {
  const int pieces = pieces_of(p);
  logprob_piece_kernel<T><<<pieces * p.rows, kThreads, 0, st>>>(p, pieces);
  const size_t smem = (size_t)pieces * p.top_k * 8;
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fta_cuda_fail(e);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.rows); cfg.blockDim = dim3(kJoin); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cfg.attrs = attr; cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, logprob_join_kernel<T>, p, pieces);
  return e == cudaSuccess ? FTA_OK : fta_cuda_fail(e);
}

}  // namespace

extern "C" int64_t fta_token_logprobs_workspace_bytes(const FtaLogprobParams* p) {
  if (int rc = check_sizes(p)) return -rc;
  return ws_bytes(*p);
}

extern "C" int fta_token_logprobs(const FtaLogprobParams* p, void* stream) {
  if (int rc = check_sizes(p)) return rc;
  if (!p->logits || !p->entropy || !p->lse || (p->n_tokens > 0 && (!p->tokens || !p->logprobs))) return FTA_E_BADARG;
  if (p->top_k > 0 && (!p->top_logprobs || !p->top_ids)) return FTA_E_BADARG;
  if (reinterpret_cast<uintptr_t>(p->logits) % (p->dtype == FTA_DTYPE_F32 ? 4 : 2) != 0) return FTA_E_BADARG;
  if (!p->workspace || (reinterpret_cast<uintptr_t>(p->workspace) & 15) || p->workspace_bytes < ws_bytes(*p)) return FTA_E_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  if (p->dtype == FTA_DTYPE_F16) return run<__half>(*p, st);
  if (p->dtype == FTA_DTYPE_BF16) return run<__nv_bfloat16>(*p, st);
  return run<float>(*p, st);
}
