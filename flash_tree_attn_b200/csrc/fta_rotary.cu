// Rotary positions of queries and keys, and the append of new tokens to the cache (include/fta.h).
//
// Angles.  A cosine needs its angle modulo one turn, and position * frequency in 32 bits has lost that
// after some 10^5 positions.  So a pair's frequency is kept as a 64-bit fraction of a turn, and
// position * fraction, modulo 2^64, IS the angle modulo one turn: an integer product, exact but for what the
// fraction is off by: 2^-52 of inv_freq / 2 pi (1 / 2 pi and the product with it are rounded in 64 bits) and
// 2^-65 of a turn.  At frequency 1 that is below 2^-23 of a turn at position 2^31, 2^-14 at 2^40.  The product's top 32
// bits, as a signed number of half-turns, go to sincospi in 24 bits: 2^-26 of a turn.
//
// What bounds it: each element is read once and written once; nothing else moves but 8 bytes per
// pair.  A block works out the cosines and sines of its tokens once, in shared memory, for all heads, while
// the first of the heads' elements are on their way.
#include "fta_common.cuh"

namespace {

constexpr int kThreads = 256;

template <typename T> __device__ __forceinline__ void unpack8(const uint4& x, float (&f)[8]) {
  const typename FtaType<T>::T2* h = reinterpret_cast<const typename FtaType<T>::T2*>(&x);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = (float)h[i].x;
    f[2 * i + 1] = (float)h[i].y;
  }
}
template <typename T> __device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(FtaType<T>::pack(f[0], f[1]), FtaType<T>::pack(f[2], f[3]), FtaType<T>::pack(f[4], f[5]), FtaType<T>::pack(f[6], f[7]));
}

// grid = (TOK tokens, sequence).  A head row is D / 16 lane tasks of two 16-byte chunks, neighbouring
// lanes taking neighbouring chunks: the two halves of 8 pairs (half), twice 4 pairs (interleaved), or
// elements that are only copied.  A head's rows of neighbouring tokens lie side by side in q, k and v.
template <typename T, bool APPEND, int TOK>
__global__ void __launch_bounds__(kThreads, 8) rotary_kernel(const FtaRotaryParams p, const int row_bits) {
  __shared__ float2 cs[TOK][128];
  __shared__ long long s_dst[2][TOK];  // where the tokens' cache rows start (K, V); -1: nowhere
  const int b = blockIdx.y, i0 = blockIdx.x * TOK;
  fta_after_previous();

  const int rot16 = p.n_freq / 8;  // lane tasks of a row that turn (half); 1 << row_bits tasks in all
  const int heads = p.H + p.Hkv + (APPEND ? p.Hkv : 0);
  const bool half = p.layout == FTA_ROTARY_HALF;
  // element offsets of task t's two chunks
  auto chunks = [&](int t, int& x0, int& x1) {
    if (half && t < rot16) {
      x0 = 8 * t;
      x1 = p.n_freq + 8 * t;
    } else {
      const int base = half ? 2 * p.n_freq : 0, u = half ? t - rot16 : t;
      x0 = base + 8 * u;
      x1 = x0 + (half ? p.D / 2 - p.n_freq : p.D / 2);
    }
  };
  // task -> head row hh (queries, then keys, then values), token and lane task
  const int tasks = (heads * TOK) << row_bits;
  uint4 a, c;
  auto read = [&](int task) {
    const int row = task >> row_bits, i = i0 + row % TOK;
    int hh = row / TOK;
    if (task >= tasks || i >= p.Q) return;
    int x0, x1;
    chunks(task & ((1 << row_bits) - 1), x0, x1);
    const T* src;
    if (hh < p.H) src = (const T*)p.q + b * p.q_sb + hh * p.q_sh + i * p.q_sq;
    else if ((hh -= p.H) < p.Hkv) src = (const T*)p.k + b * p.k_sb + hh * p.k_sh + i * p.k_sq;
    else src = (const T*)p.v + b * p.v_sb + (hh - p.Hkv) * p.v_sh + i * p.v_sq;
    a = *reinterpret_cast<const uint4*>(src + x0);
    c = *reinterpret_cast<const uint4*>(src + x1);
  };
  read(threadIdx.x);

  const int L = APPEND ? fta_load_len(p.kv_seq_len, p.len_is_i64, b, p.ctx) : 0;
  if (APPEND && (int)threadIdx.x < TOK) {
    const unsigned wide = (unsigned)L + i0 + threadIdx.x;  // a long cache and a long chunk: past 2^31, below 2^32
    bool fits = wide < (unsigned)p.ctx;
    const int row = fits ? (int)wide : 0;
    long long at = b, in = row;
    if (p.block_table != nullptr && fits) {
      at = p.block_table[b * p.bt_sb + row / p.page_size];
      in = row % p.page_size;
      fits = at >= 0 && at < p.n_pages;
    }
    s_dst[0][threadIdx.x] = fits ? at * p.kc_sb + in * p.kc_st : -1;
    s_dst[1][threadIdx.x] = fits ? at * p.vc_sb + in * p.vc_st : -1;
  }
  for (int j = threadIdx.x; j < p.n_freq * TOK; j += kThreads) {
    const int tok = j / p.n_freq, f = j - tok * p.n_freq, i = i0 + tok;
    if (i >= p.Q) break;
    long long pos = APPEND ? L : 0;
    if (p.positions != nullptr) {
      const long long at = b * p.pos_sb + i * p.pos_sq;
      pos = p.pos_is_i64 ? reinterpret_cast<const long long*>(p.positions)[at] : reinterpret_cast<const int*>(p.positions)[at];
    }
    pos += p.offsets != nullptr ? p.offsets[i] : (p.positions == nullptr || p.pos_sq == 0 ? i : 0);
    const double turns = p.inv_freq[f] * 0.15915494309189535;  // 1 / (2 pi)
    const unsigned long long step = __double2ull_rn((turns - floor(turns)) * 18446744073709551616.0);
    unsigned long long phase = (unsigned long long)pos * step;
    if (p.inverse) phase = 0ull - phase;
    float sn, cn;
    sincospif((float)(int)(phase >> 32) * 4.656612873077393e-10f, &sn, &cn);  // 2^-31: half-turns
    cs[tok][f] = make_float2(cn * p.amplitude, sn * p.amplitude);
  }
  // one block per sequence: nobody else reads the length, and everybody here has
  __syncthreads();
  if (APPEND && gridDim.x == 1 && threadIdx.x == 0) {
    const int to = (int)min((long long)L + p.Q, (long long)p.ctx);
    if (p.len_is_i64) reinterpret_cast<long long*>(p.kv_seq_len)[b] = to;
    else reinterpret_cast<int*>(p.kv_seq_len)[b] = to;
  }

  // eight blocks an SM keep enough rows in flight: two tasks a thread at once, with five blocks, took as long
  for (int task = threadIdx.x; task < tasks; task += kThreads) {
    if (task != (int)threadIdx.x) read(task);
    const int row = task >> row_bits, t = task & ((1 << row_bits) - 1);
    const int tok = row % TOK, i = i0 + tok, hh = row / TOK;
    if (i >= p.Q) continue;
    int x0, x1;
    chunks(t, x0, x1);
    if (hh < p.H + p.Hkv && (half ? t < rot16 : x0 < 2 * p.n_freq)) {
      float y[8], z[8];
      unpack8<T>(a, y);
      unpack8<T>(c, z);
      if (half) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 f = cs[tok][8 * t + e];
          const float n = y[e] * f.x - z[e] * f.y;
          z[e] = z[e] * f.x + y[e] * f.y;
          y[e] = n;
        }
      } else {
        const bool both = x1 < 2 * p.n_freq;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = cs[tok][x0 / 2 + e];
          const float n = y[2 * e] * f.x - y[2 * e + 1] * f.y;
          y[2 * e + 1] = y[2 * e + 1] * f.x + y[2 * e] * f.y;
          y[2 * e] = n;
          if (both) {
            const float2 g = cs[tok][x1 / 2 + e];
            const float n1 = z[2 * e] * g.x - z[2 * e + 1] * g.y;
            z[2 * e + 1] = z[2 * e + 1] * g.x + z[2 * e] * g.y;
            z[2 * e] = n1;
          }
        }
      }
      a = pack8<T>(y);
      c = pack8<T>(z);
    }
    T* dst;
    if (hh < p.H) {
      dst = (T*)p.q_out + (((long long)b * p.H + hh) * p.Q + i) * p.D;
    } else if (!APPEND) {
      dst = (T*)p.k_out + (((long long)b * p.Hkv + hh - p.H) * p.Q + i) * p.D;
    } else {
      const bool v = hh >= p.H + p.Hkv;
      const long long at = s_dst[v][tok];
      if (at < 0) continue;
      dst = v ? (T*)p.v_cache + at + (hh - p.H - p.Hkv) * p.vc_sh : (T*)p.k_cache + at + (hh - p.H) * p.kc_sh;
    }
    *reinterpret_cast<uint4*>(dst + x0) = a;
    *reinterpret_cast<uint4*>(dst + x1) = c;
  }
}

__global__ void grow_lengths_kernel(const FtaRotaryParams p) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  fta_after_previous();  // every block of the append has read the lengths
  if (b >= p.B) return;
  const long long L = fta_load_len(p.kv_seq_len, p.len_is_i64, b, p.ctx) + (long long)p.Q;
  const int to = (int)(L < p.ctx ? L : p.ctx);
  if (p.len_is_i64) reinterpret_cast<long long*>(p.kv_seq_len)[b] = to;
  else reinterpret_cast<int*>(p.kv_seq_len)[b] = to;
}

bool aligned16(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }
bool rows16(const void* x, int64_t a, int64_t b, int64_t c) { return aligned16(x) && a % 8 == 0 && b % 8 == 0 && c % 8 == 0; }

int check(const FtaRotaryParams* p, bool append) {
  if (!p || p->B <= 0 || p->H < 0 || p->Hkv < 0 || p->H + p->Hkv <= 0 || p->Q <= 0) return FTA_E_BADARG;
  if (p->D != 32 && p->D != 64 && p->D != 128 && p->D != 256) return FTA_E_BADARG;
  if (p->dtype != FTA_DTYPE_F16 && p->dtype != FTA_DTYPE_BF16) return FTA_E_BADARG;
  // 16-byte chunks hold whole halves of 8 pairs
  if (p->n_freq < 0 || p->n_freq % 8 != 0 || 2 * p->n_freq > p->D || (p->n_freq > 0 && !p->inv_freq)) return FTA_E_BADARG;
  if (p->layout != FTA_ROTARY_HALF && p->layout != FTA_ROTARY_INTERLEAVED) return FTA_E_BADARG;
  if (p->B > 65535) return FTA_E_UNSUPPORTED;
  if (p->H > 0 && (!p->q || !p->q_out || !rows16(p->q, p->q_sb, p->q_sh, p->q_sq) || !aligned16(p->q_out))) return FTA_E_BADARG;
  if (p->Hkv > 0 && (!p->k || !rows16(p->k, p->k_sb, p->k_sh, p->k_sq))) return FTA_E_BADARG;
  if (!append) return p->n_freq == 0 || !p->positions || (p->Hkv > 0 && (!p->k_out || !aligned16(p->k_out))) ? FTA_E_BADARG : FTA_OK;
  if (p->Hkv <= 0 || p->ctx < 0 || !p->v || !p->k_cache || !p->v_cache || !p->kv_seq_len) return FTA_E_BADARG;
  if (!rows16(p->v, p->v_sb, p->v_sh, p->v_sq) || !rows16(p->k_cache, p->kc_sb, p->kc_sh, p->kc_st) ||
      !rows16(p->v_cache, p->vc_sb, p->vc_sh, p->vc_st))
    return FTA_E_BADARG;
  if (p->block_table && (p->page_size < 1 || p->n_pages < 1 || p->bt_sb < 0 || (p->B > 1 && (long long)p->bt_sb * p->page_size < p->ctx)))
    return FTA_E_BADARG;
  return FTA_OK;
}

template <bool APPEND>
int launch(const FtaRotaryParams* p, cudaStream_t st) {
  if (int rc = check(p, APPEND)) return rc;
  // Four tokens a block once that still leaves every SM several blocks: they share the start of a block
  // (length, page, a barrier) and a head's rows of four tokens are one piece of memory.
  const bool four = p->Q >= 4 && (long long)p->B * p->Q >= kFtaSms * 16;
  const dim3 grid(four ? (p->Q + 3) / 4 : p->Q, p->B);
  const int bits = p->D == 32 ? 1 : p->D == 64 ? 2 : p->D == 128 ? 3 : 4;
  const bool f16 = p->dtype == FTA_DTYPE_F16;
  cudaError_t e;
  if (four && f16) e = fta_launch_after(rotary_kernel<__half, APPEND, 4>, grid, kThreads, 0, st, 1, *p, bits);
  else if (four) e = fta_launch_after(rotary_kernel<__nv_bfloat16, APPEND, 4>, grid, kThreads, 0, st, 1, *p, bits);
  else if (f16) e = fta_launch_after(rotary_kernel<__half, APPEND, 1>, grid, kThreads, 0, st, 1, *p, bits);
  else e = fta_launch_after(rotary_kernel<__nv_bfloat16, APPEND, 1>, grid, kThreads, 0, st, 1, *p, bits);
  if (APPEND && grid.x > 1 && e == cudaSuccess) e = fta_launch_after(grow_lengths_kernel, dim3((p->B + 127) / 128), 128, 0, st, 1, *p);
  return e == cudaSuccess ? FTA_OK : fta_cuda_fail(e);
}

}  // namespace

extern "C" int fta_apply_rotary(const FtaRotaryParams* p, void* stream) { return launch<false>(p, (cudaStream_t)stream); }
extern "C" int fta_append_tokens(const FtaRotaryParams* p, void* stream) { return launch<true>(p, (cudaStream_t)stream); }
