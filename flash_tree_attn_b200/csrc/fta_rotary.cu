// Rotary positions of queries and keys, and the append of new tokens to the cache (include/fta.h).
//
// Angles.  A cosine needs its angle modulo one turn, and position * frequency in 32 bits has lost that
// after some 10^5 positions.  So a pair's frequency is kept as a 64-bit fraction of a turn, and
// position * fraction, modulo 2^64, IS the angle modulo one turn: an integer product, exact but for
// the fraction's own rounding (2^-64 turns a position).  Its top 32 bits, as a signed number of
// half-turns, go to sincospi.
//
// What bounds it: each element is read once and written once; nothing else moves but 8 bytes per
// pair.  A block works out the cosines and sines of its tokens once, in shared memory, for all heads.
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

// grid = (token, sequence).  A head row is D / 16 lane tasks of two 16-byte chunks: the two halves of 8
// pairs (or 8 adjacent pairs), or 16 elements that are only copied.
template <typename T, bool APPEND>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const FtaRotaryParams p) {
  __shared__ float2 cs[128];
  const int i = blockIdx.x, b = blockIdx.y;
  const int L = APPEND ? fta_load_len(p.kv_seq_len, p.len_is_i64, b, p.ctx) : 0;
  if ((int)threadIdx.x < p.n_freq) {
    long long pos = APPEND ? L : 0;
    if (p.positions != nullptr) {
      const long long at = b * p.pos_sb + i * p.pos_sq;
      pos = p.pos_is_i64 ? reinterpret_cast<const long long*>(p.positions)[at] : reinterpret_cast<const int*>(p.positions)[at];
    }
    pos += p.offsets != nullptr ? p.offsets[i] : (p.positions == nullptr || p.pos_sq == 0 ? i : 0);
    const double turns = p.inv_freq[threadIdx.x] * 0.15915494309189535;  // 1 / (2 pi)
    const unsigned long long step = __double2ull_rn((turns - floor(turns)) * 18446744073709551616.0);
    unsigned long long phase = (unsigned long long)pos * step;
    if (p.inverse) phase = 0ull - phase;
    float s, c;
    sincospif((float)(int)(phase >> 32) * 4.656612873077393e-10f, &s, &c);  // 2^-31: half-turns
    cs[threadIdx.x] = make_float2(c * p.amplitude, s * p.amplitude);
  }
  // one block per sequence: nobody else reads the length, and everybody here has
  __syncthreads();
  if (APPEND && gridDim.x == 1 && threadIdx.x == 0) {
    const int to = (int)min((long long)L + p.Q, (long long)p.ctx);
    if (p.len_is_i64) reinterpret_cast<long long*>(p.kv_seq_len)[b] = to;
    else reinterpret_cast<int*>(p.kv_seq_len)[b] = to;
  }

  const int per_row = p.D / 16, rot16 = p.n_freq / 8;  // lane tasks of a row, those that turn
  const int heads = p.H + p.Hkv + (APPEND ? p.Hkv : 0);
  long long kdst = 0, vdst = 0;  // where the cache row starts
  bool fits = true;
  if (APPEND) {
    const int row = L + i;
    long long at = b, r = row;
    fits = row >= 0 && row < p.ctx;
    if (p.block_table != nullptr && fits) {
      at = p.block_table[b * p.bt_sb + row / p.page_size];
      r = row % p.page_size;
      fits = at >= 0 && at < p.n_pages;
    }
    kdst = at * p.kc_sb + r * p.kc_st;
    vdst = at * p.vc_sb + r * p.vc_st;
  }
  for (int task = threadIdx.x; task < heads * per_row; task += kThreads) {
    const int hh = task / per_row, t = task - hh * per_row;
    const T* src;
    T* dst;
    bool turn = t < rot16;
    if (hh < p.H) {
      src = (const T*)p.q + b * p.q_sb + hh * p.q_sh + i * p.q_sq;
      dst = (T*)p.q_out + (((long long)b * p.H + hh) * p.Q + i) * p.D;
    } else if (hh < p.H + p.Hkv) {
      const int h = hh - p.H;
      src = (const T*)p.k + b * p.k_sb + h * p.k_sh + i * p.k_sq;
      dst = APPEND ? (T*)p.k_cache + kdst + h * p.kc_sh : (T*)p.k_out + (((long long)b * p.Hkv + h) * p.Q + i) * p.D;
      if (!fits) continue;
    } else {
      const int h = hh - p.H - p.Hkv;
      src = (const T*)p.v + b * p.v_sb + h * p.v_sh + i * p.v_sq;
      dst = (T*)p.v_cache + vdst + h * p.vc_sh;
      turn = false;
      if (!fits) continue;
    }
    const bool halves = p.layout == FTA_ROTARY_HALF && t < rot16;  // v included: the same chunks, copied
    const int x0 = halves ? 8 * t : 16 * t, x1 = halves ? p.n_freq + 8 * t : 16 * t + 8;
    uint4 a = *reinterpret_cast<const uint4*>(src + x0), c = *reinterpret_cast<const uint4*>(src + x1);
    if (turn) {
      float u[8], w[8];
      unpack8<T>(a, u);
      unpack8<T>(c, w);
      if (p.layout == FTA_ROTARY_HALF) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 f = cs[8 * t + e];
          const float y = u[e] * f.x - w[e] * f.y;
          w[e] = w[e] * f.x + u[e] * f.y;
          u[e] = y;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 f = cs[8 * t + e];
          float* z = e < 4 ? u + 2 * e : w + 2 * (e - 4);
          const float y = z[0] * f.x - z[1] * f.y;
          z[1] = z[1] * f.x + z[0] * f.y;
          z[0] = y;
        }
      }
      a = pack8<T>(u);
      c = pack8<T>(w);
    }
    *reinterpret_cast<uint4*>(dst + x0) = a;
    *reinterpret_cast<uint4*>(dst + x1) = c;
  }
}

__global__ void grow_lengths_kernel(const FtaRotaryParams p) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
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
  const dim3 grid(p->Q, p->B);
  if (p->dtype == FTA_DTYPE_F16) rotary_kernel<__half, APPEND><<<grid, kThreads, 0, st>>>(*p);
  else rotary_kernel<__nv_bfloat16, APPEND><<<grid, kThreads, 0, st>>>(*p);
  if (APPEND && p->Q > 1) grow_lengths_kernel<<<(p->B + 127) / 128, 128, 0, st>>>(*p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FTA_OK : fta_cuda_fail(e);
}

}  // namespace

extern "C" int fta_apply_rotary(const FtaRotaryParams* p, void* stream) { return launch<false>(p, (cudaStream_t)stream); }
extern "C" int fta_append_tokens(const FtaRotaryParams* p, void* stream) { return launch<true>(p, (cudaStream_t)stream); }
