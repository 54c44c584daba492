// Eviction of cache rows by accumulated attention weight (include/fta.h: fta_evict_rows).
//
// Select: one block per (sequence, KV head) finds the smallest weight that is kept by a radix select
// over the weights' ordered bits (four passes of 8 bits), then walks the rows once more in order and
// writes the list of kept rows, moving their weights up as it goes.
// Move: new row i takes old row kept[i] >= i.  A block owns a column slice of one head's K or V and
// walks the list in chunks: all of a chunk's rows are read, then written.  A write goes to rows below
// the chunk's end, a later chunk's rows lie at or above it, so reads never see a write.
//
// What bounds it: the kept rows of K and V are read and written once (8 D bytes a row); the weights
// are small against that.
#include "fta_common.cuh"

namespace {

constexpr int kSelect = 1024;
constexpr int kMove = 256;
constexpr int kAhead = 4;  // rows in flight per thread

// order of floats as unsigned integers; -0 and +0 alike, NaN on top
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x);
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (b == 0x80000000u) return b;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__global__ void __launch_bounds__(kSelect) evict_select_kernel(const FtaEvictParams p) {
  __shared__ int hist[256];
  __shared__ int s_bin, s_left;
  __shared__ int s_warp[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x - b * p.Hkv;
  const int L = fta_load_len(p.kv_seq_len, p.len_is_i64, b, p.ctx);
  int* kept = p.kept + (long long)blockIdx.x * p.budget;
  if (L <= p.budget) {
    for (int i = tid; i < p.budget; i += kSelect) kept[i] = i < L ? i : -1;
    return;
  }
  float* w = p.row_weights + b * p.rw_sb + h * p.rw_sh;
  const int n = L - p.recent, want = p.budget - p.recent;  // n > want

  // the want-th largest of w[0, n): its bits from the top, `left` counts down to its rank among equals
  uint32_t prefix = 0, mask = 0;
  int left = want;
  if (want > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kSelect) hist[i] = 0;
      __syncthreads();
      for (int r = tid; r < n; r += kSelect) {
        const uint32_t k = ordered(w[r]);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      if (warp == 0) {  // lane holds bins 8 lane .. 8 lane + 7; bins above it come first
        int mine = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) mine += hist[8 * lane + i];
        int above = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int t = __shfl_down_sync(0xffffffffu, above, o);
          if (lane + o < 32) above += t;
        }
        above -= mine;
        if (above < left && left <= above + mine) {
          int rest = left - above, i = 7;
          while (rest > hist[8 * lane + i]) rest -= hist[8 * lane + i--];
          s_bin = 8 * lane + i;
          s_left = rest;
        }
      }
      __syncthreads();
      prefix |= (uint32_t)s_bin << shift;
      mask |= 255u << shift;
      left = s_left;
      __syncthreads();
    }
  }

  // in order: larger ones, and the first `left` equal ones
  int taken = 0, equal = 0;  // kept so far, equal ones seen so far
  for (int base = 0; base < n && want > 0; base += kSelect) {
    const int r = base + tid;
    const float x = r < n ? w[r] : 0.f;
    const uint32_t k = ordered(x);
    const bool eq = r < n && k == prefix, gt = r < n && k > prefix;
    const unsigned eqs = __ballot_sync(0xffffffffu, eq), gts = __ballot_sync(0xffffffffu, gt);
    if (lane == 0) { s_warp[0][warp] = __popc(eqs); s_warp[1][warp] = __popc(gts); }
    __syncthreads();
    int e = s_warp[0][lane], g = s_warp[1][lane];  // 32 warps: inclusive sums over them
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int te = __shfl_up_sync(0xffffffffu, e, o), tg = __shfl_up_sync(0xffffffffu, g, o);
      if (lane >= o) { e += te; g += tg; }
    }
    const int e_all = __shfl_sync(0xffffffffu, e, 31), g_all = __shfl_sync(0xffffffffu, g, 31);
    const int e_before = warp == 0 ? 0 : __shfl_sync(0xffffffffu, e, (warp - 1) & 31);
    const int g_before = warp == 0 ? 0 : __shfl_sync(0xffffffffu, g, (warp - 1) & 31);
    const unsigned below = (1u << lane) - 1;
    const int my_eq = equal + e_before + __popc(eqs & below);  // equal ones before this row
    const int my_gt = g_before + __popc(gts & below);
    if (gt || (eq && my_eq < left)) {
      const int at = taken + my_gt + min(my_eq, left) - min(equal, left);
      kept[at] = r;
      w[at] = x;  // at <= r, and every row of this chunk has been read
    }
    taken += g_all + min(equal + e_all, left) - min(equal, left);
    equal += e_all;
    __syncthreads();
  }
  // the recent rows move up behind them
  for (int base = 0; base < p.recent; base += kSelect) {
    const int i = base + tid;
    const float x = i < p.recent ? w[n + i] : 0.f;
    __syncthreads();
    if (i < p.recent) {
      kept[want + i] = n + i;
      w[want + i] = x;
    }
  }
  __syncthreads();
  for (int r = p.budget + tid; r < L; r += kSelect) w[r] = 0.f;
}

// grid = (B * Hkv, K or V, column slices); a row of a slice is `chunks` 16-byte chunks
__global__ void __launch_bounds__(kMove) evict_move_kernel(const FtaEvictParams p, const int chunks) {
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x - b * p.Hkv;
  const int* kept = p.kept + (long long)blockIdx.x * p.budget;
  if (blockIdx.y == 0 && blockIdx.z == 0 && h == 0 && threadIdx.x == 0) {
    // the select kernel has read the lengths, and this one does not
    const int L = min(fta_load_len(p.kv_seq_len, p.len_is_i64, b, p.ctx), p.budget);
    if (p.len_is_i64) reinterpret_cast<long long*>(p.kv_seq_len)[b] = L;
    else reinterpret_cast<int*>(p.kv_seq_len)[b] = L;
  }
  // kept[i] - i never falls: rows before the first moved one stay where they are
  int lo = 0, hi = p.budget;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    const int r = kept[mid];
    if (r > mid) hi = mid; else lo = mid + 1;
  }
  const long long sb = blockIdx.y ? p.v_sb : p.k_sb, sh = blockIdx.y ? p.v_sh : p.k_sh, st = blockIdx.y ? p.v_st : p.k_st;
  uint16_t* cache = (uint16_t*)(blockIdx.y ? p.v_cache : p.k_cache) + h * sh + (long long)blockIdx.z * chunks * 8;
  auto row_at = [&](int r) -> uint4* {
    long long at = b;
    if (p.block_table != nullptr) {
      at = p.block_table[b * p.bt_sb + r / p.page_size];
      if (at < 0 || at >= p.n_pages) return nullptr;
      r %= p.page_size;
    }
    return reinterpret_cast<uint4*>(cache + at * sb + (long long)r * st);
  };
  const int per = kMove / chunks, mine = threadIdx.x / chunks, c = threadIdx.x - mine * chunks;
  for (int base = lo; base < p.budget; base += per * kAhead) {
    uint4 x[kAhead];
    bool got[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = base + u * per + mine;
      const uint4* src = i < p.budget && kept[i] >= 0 ? row_at(kept[i]) : nullptr;
      got[u] = src != nullptr;
      if (got[u]) x[u] = src[c];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      uint4* dst = got[u] ? row_at(base + u * per + mine) : nullptr;
      if (dst != nullptr) dst[c] = x[u];
    }
  }
}

bool rows16(const void* x, int64_t a, int64_t b, int64_t c) {
  return (reinterpret_cast<uintptr_t>(x) & 15) == 0 && a % 8 == 0 && b % 8 == 0 && c % 8 == 0;
}

}  // namespace

extern "C" int fta_evict_rows(const FtaEvictParams* p, void* stream) {
  if (!p || p->B <= 0 || p->Hkv <= 0 || p->ctx < 0 || p->budget <= 0 || p->recent < 0 || p->recent > p->budget) return FTA_E_BADARG;
  if (p->D != 32 && p->D != 64 && p->D != 128 && p->D != 256) return FTA_E_BADARG;
  if (!p->k_cache || !p->v_cache || !p->kv_seq_len || !p->row_weights || !p->kept) return FTA_E_BADARG;
  if (!rows16(p->k_cache, p->k_sb, p->k_sh, p->k_st) || !rows16(p->v_cache, p->v_sb, p->v_sh, p->v_st)) return FTA_E_BADARG;
  if (p->block_table && (p->page_size < 1 || p->n_pages < 1 || p->bt_sb < 0 || (p->B > 1 && (long long)p->bt_sb * p->page_size < p->ctx)))
    return FTA_E_BADARG;
  cudaStream_t st = (cudaStream_t)stream;
  evict_select_kernel<<<p->B * p->Hkv, kSelect, 0, st>>>(*p);
  // column slices until there are blocks for every SM; no slice below a 32-byte sector
  int slices = 1;
  while ((long long)p->B * p->Hkv * 2 * slices < 2 * 148 && p->D / 8 / slices > 2) slices *= 2;
  evict_move_kernel<<<dim3(p->B * p->Hkv, 2, slices), kMove, 0, st>>>(*p, p->D / 8 / slices);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? FTA_OK : fta_cuda_fail(e);
}
