// Eviction of cache rows by accumulated attention weight (include/fta.h: fta_evict_rows).
//
// Select: one block per (sequence, KV head) finds the smallest weight that is kept by a radix select
// over the weights' ordered bits, held in shared memory, counts the kept rows of each warp's stretch, and
// writes the list of kept rows and their weights in order.  Digits are 11, 11 and 10 bits wide: the top
// 11 are the exponent and two bits more, over which weights spread; with 8 bits most of a warp's
// counts met in the same few bins, one after the other.
// Move: new row i takes old row kept[i] >= i.  A block, or a cluster of them, owns a column slice of one
// head's K or V and walks the list in chunks: all of a chunk's rows are read, then written.  A write goes to rows below
// the chunk's end, a later chunk's rows lie at or above it, so reads never see a write, and the next
// chunk's reads are under way while this one's rows are written.
//
// What bounds it: the kept rows of K and V are read and written once (8 D bytes a row); the weights
// are small against that.
#include <cooperative_groups.h>

#include "fta_common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kSelect = 1024;
constexpr int kKeys = 24 * 1024;  // rows whose weights fit the select block's shared memory (two blocks an SM)
constexpr int kMove = 256;
constexpr int kAhead = 3;         // rows per thread and chunk
constexpr int kBins = 2048;
constexpr int kMostRows = FTA_MAX_ROWS;  // loops over rows are 32-bit and step past the end by up to 2^15

// Weights are handled as their bits throughout: arithmetic would take the smallest ones for zeros.
// Their order as unsigned integers; -0 and +0 alike, NaN on top.
__device__ __forceinline__ uint32_t ordered(uint32_t b) {
  if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (b == 0x80000000u) return b;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Moves w[from, from + n) to w[to, to + n), to <= from: a chunk is read, then written.
template <typename F> __device__ __forceinline__ void move_up(uint32_t* w, int to, int n, F&& from) {
  for (int base = 0; base < n; base += 4 * kSelect) {
    uint32_t x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = base + u * kSelect + (int)threadIdx.x;
      x[u] = i < n ? w[from(i)] : 0u;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = base + u * kSelect + (int)threadIdx.x;
      if (i < n) w[to + i] = x[u];
    }
  }
}

// `room`: weights that the dynamic shared memory holds; a longer sequence's are read again in every pass
__global__ void __launch_bounds__(kSelect) evict_select_kernel(const FtaEvictParams p, const int room) {
  extern __shared__ __align__(16) uint32_t s_w[];
  __shared__ int hist[kBins];
  __shared__ int s_bin, s_left;
  __shared__ int s_equal[32], s_larger[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x - b * p.Hkv;
  fta_after_previous();
  const int L = fta_load_len(p.kv_seq_len, p.len_is_i64, b, p.ctx);
  int* kept = p.kept + (long long)blockIdx.x * p.budget;
  if (L <= p.budget) {
    for (int i = tid; i < p.budget; i += kSelect) kept[i] = i < L ? i : -1;
    return;
  }
  uint32_t* w = reinterpret_cast<uint32_t*>(p.row_weights) + b * p.rw_sb + h * p.rw_sh;
  const int n = L - p.recent, want = p.budget - p.recent;  // n > want

  if (want > 0) {
    const bool held = n <= room;
    if (held) {
#pragma unroll 8
      for (int r = tid; r < n; r += kSelect) s_w[r] = w[r];
    }
    // the keys of rows r .. r + 3, r a multiple of 4; 0, which is below every weight, past the end
    auto keys = [&](int r, uint32_t (&k)[4]) {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (held) {
        if (r < n) x = *reinterpret_cast<const uint4*>(s_w + r);  // n <= room, a multiple of 4
      } else {
        if (r < n) x.x = w[r];
        if (r + 1 < n) x.y = w[r + 1];
        if (r + 2 < n) x.z = w[r + 2];
        if (r + 3 < n) x.w = w[r + 3];
      }
      k[0] = r < n ? ordered(x.x) : 0u;
      k[1] = r + 1 < n ? ordered(x.y) : 0u;
      k[2] = r + 2 < n ? ordered(x.z) : 0u;
      k[3] = r + 3 < n ? ordered(x.w) : 0u;
    };

    // the want-th largest of w[0, n): its bits from the top, `left` counts down to its rank among equals
    uint32_t prefix = 0, mask = 0;
    int left = want;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, digit = pass < 2 ? 2047 : 1023;
      hist[tid] = 0;
      hist[tid + kSelect] = 0;
      __syncthreads();
      for (int r = 4 * tid; r < n; r += 4 * kSelect) {
        uint32_t k[4];
        keys(r, k);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((k[e] & mask) == prefix && k[e] != 0u) atomicAdd(&hist[(k[e] >> shift) & digit], 1);
      }
      __syncthreads();
      // a thread holds bins 2047 - 2 tid and the one below; `above` counts the bins that come before
      const int bin = kBins - 1 - 2 * tid, first = hist[bin], mine = first + hist[bin - 1];
      int above = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, above, o);
        if (lane >= o) above += t;
      }
      if (lane == 31) s_equal[warp] = above;
      __syncthreads();
      above += __reduce_add_sync(0xffffffffu, lane < warp ? s_equal[lane] : 0) - mine;
      if (above < left && left <= above + mine) {
        const bool upper = left <= above + first;
        s_bin = upper ? bin : bin - 1;
        s_left = left - above - (upper ? 0 : first);
      }
      __syncthreads();
      prefix |= (uint32_t)s_bin << shift;
      mask |= (uint32_t)digit << shift;
      left = s_left;
    }

    // Larger ones are kept, and the first `left` equal ones.  Each warp counts both in a stretch of rows,
    // then, knowing what lies before it, writes its part of the list.
    const int per = fta_cdiv(fta_cdiv(n, 32), 128) * 128, r0 = warp * per, r1 = min(n, r0 + per);
    int equal = 0, larger = 0;
    for (int r = r0 + 4 * lane; r < r1; r += 128) {
      uint32_t k[4];
      keys(r, k);
#pragma unroll
      for (int e = 0; e < 4; ++e) { equal += k[e] == prefix; larger += k[e] > prefix; }
    }
    equal = __reduce_add_sync(0xffffffffu, equal);
    larger = __reduce_add_sync(0xffffffffu, larger);
    __syncthreads();  // s_equal of the last pass has been read
    if (lane == 0) { s_equal[warp] = equal; s_larger[warp] = larger; }
    __syncthreads();
    equal = __reduce_add_sync(0xffffffffu, lane < warp ? s_equal[lane] : 0);
    larger = __reduce_add_sync(0xffffffffu, lane < warp ? s_larger[lane] : 0);
    for (int first = r0; first < r1; first += 128) {
      const int r = first + 4 * lane;
      uint32_t k[4];
      keys(r, k);
      int both = 0;  // equal ones in the low half, larger ones in the high half
#pragma unroll
      for (int e = 0; e < 4; ++e) both += (k[e] == prefix ? 1 : 0) + (k[e] > prefix ? 1 << 16 : 0);
      int sum = both;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += t;
      }
      int e_before = equal + ((sum - both) & 0xffff), g_before = larger + ((sum - both) >> 16);
      const int all = __shfl_sync(0xffffffffu, sum, 31);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (k[e] > prefix || (k[e] == prefix && e_before < left)) {
          const int at = g_before + min(e_before, left);
          kept[at] = r + e;
          if (held) w[at] = s_w[r + e];  // nobody reads w[0, n) any more
        }
        e_before += k[e] == prefix;
        g_before += k[e] > prefix;
      }
      equal += all & 0xffff;
      larger += all >> 16;
    }
    __syncthreads();
    if (!held) move_up(w, 0, want, [&](int i) { return kept[i]; });
  }
  for (int i = tid; i < p.recent; i += kSelect) kept[want + i] = n + i;
  move_up(w, want, p.recent, [&](int i) { return n + i; });
  __syncthreads();
  for (int r = p.budget + tid; r < L; r += kSelect) w[r] = 0u;
}

// grid = (B * Hkv * blocks of a cluster, K or V, column slices); a row of a slice is `chunks` 16-byte chunks
__global__ void __launch_bounds__(kMove, 4) evict_move_kernel(const FtaEvictParams p, const int chunks, const int blocks) {
  const int unit = blockIdx.x / blocks, rank = blockIdx.x - unit * blocks;
  const int b = unit / p.Hkv, h = unit - b * p.Hkv;
  const int* kept = p.kept + (long long)unit * p.budget;
  fta_after_previous();
  if (rank == 0 && blockIdx.y == 0 && blockIdx.z == 0 && h == 0 && threadIdx.x == 0) {
    // the select kernel has read the lengths, and this one does not
    const int L = min(fta_load_len(p.kv_seq_len, p.len_is_i64, b, p.ctx), p.budget);
    if (p.len_is_i64) reinterpret_cast<long long*>(p.kv_seq_len)[b] = L;
    else reinterpret_cast<int*>(p.kv_seq_len)[b] = L;
  }
  // kept[i] - i never falls: rows before the first moved one stay where they are.  Each step of the search
  // probes kMove places at once.
  int lo = 0, hi = p.budget;
  while (lo < hi) {
    const int step = fta_cdiv(hi - lo, kMove), i = lo + (int)threadIdx.x * step;
    const int stay = __syncthreads_count(i < hi && kept[i] <= i);  // probes 0 .. stay - 1 stay
    if (stay == 0) break;  // lo itself moves
    const int from = lo + (stay - 1) * step + 1;
    hi = min(hi, from - 1 + step);  // the next probe moves, or lies at the end
    lo = from;
  }
  const long long sb = blockIdx.y ? p.v_sb : p.k_sb, sh = blockIdx.y ? p.v_sh : p.k_sh, st = blockIdx.y ? p.v_st : p.k_st;
  const int per = kMove / chunks * blocks, mine = kMove / chunks * rank + threadIdx.x / chunks, c = threadIdx.x % chunks;
  uint16_t* cache = (uint16_t*)(blockIdx.y ? p.v_cache : p.k_cache) + h * sh + ((long long)blockIdx.z * chunks + c) * 8;
  const int page_bits = (p.page_size & (p.page_size - 1)) == 0 ? __ffs(p.page_size) - 1 : -1;  // a division costs as much as a row's copy
  const int* table = p.block_table + b * p.bt_sb;
  auto row_at = [&](int r) -> uint4* {
    long long at = b;
    if (p.block_table != nullptr) {
      const int slot = page_bits >= 0 ? r >> page_bits : r / p.page_size;
      at = table[slot];
      if (at < 0 || at >= p.n_pages) return nullptr;
      r -= slot * p.page_size;
    }
    return reinterpret_cast<uint4*>(cache + at * sb + (long long)r * st);
  };
  // three stages: which rows (two chunks ahead), their contents (one ahead), the writes
  int rows[kAhead];
  uint4 now[kAhead], next[kAhead];
  unsigned has_now = 0, has_next = 0;
  auto ask = [&](int base) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = base + u * per + mine;
      rows[u] = i < p.budget ? kept[i] : -1;
    }
  };
  auto read = [&](uint4 (&x)[kAhead]) {
    unsigned has = 0;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint4* src = rows[u] >= 0 ? row_at(rows[u]) : nullptr;
      if (src != nullptr) { x[u] = *src; has |= 1u << u; }
    }
    return has;
  };
  const int chunk = per * kAhead;
  if (lo >= p.budget) return;
  ask(lo);
  has_now = read(now);
  ask(lo + chunk);
  for (int base = lo; base < p.budget; base += chunk) {
    has_next = read(next);
    ask(base + 2 * chunk);
    if (blocks == 1) __syncthreads();  // everybody has read this chunk
    else cg::this_cluster().sync();
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      uint4* dst = (has_now >> u) & 1 ? row_at(base + u * per + mine) : nullptr;
      if (dst != nullptr) *dst = now[u];
      now[u] = next[u];
    }
    has_now = has_next;
  }
}

bool rows16(const void* x, int64_t a, int64_t b, int64_t c) {
  return (reinterpret_cast<uintptr_t>(x) & 15) == 0 && a % 8 == 0 && b % 8 == 0 && c % 8 == 0;
}

}  // namespace

extern "C" int fta_evict_rows(const FtaEvictParams* p, void* stream) {
  if (!p || p->B <= 0 || p->Hkv <= 0 || p->ctx < 0 || p->budget <= 0 || p->recent < 0 || p->recent > p->budget) return FTA_E_BADARG;
  if (p->D != 32 && p->D != 64 && p->D != 128 && p->D != 256) return FTA_E_BADARG;
  if (p->ctx > kMostRows || p->budget > kMostRows) return FTA_E_UNSUPPORTED;
  if (!p->k_cache || !p->v_cache || !p->kv_seq_len || !p->row_weights || !p->kept) return FTA_E_BADARG;
  if (!rows16(p->k_cache, p->k_sb, p->k_sh, p->k_st) || !rows16(p->v_cache, p->v_sb, p->v_sh, p->v_st)) return FTA_E_BADARG;
  if (p->block_table && (p->page_size < 1 || p->n_pages < 1 || p->bt_sb < 0 || (p->B > 1 && (long long)p->bt_sb * p->page_size < p->ctx)))
    return FTA_E_BADARG;
  cudaStream_t st = (cudaStream_t)stream;
  static unsigned long long configured = 0ull;  // per device: the opt-in shared-memory limit is set
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return fta_cuda_fail(e);
  if (!((configured >> (dev & 63)) & 1ull)) {
    e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kKeys * 4);
    if (e != cudaSuccess) return fta_cuda_fail(e);
    configured |= 1ull << (dev & 63);
  }
  const int room = p->ctx < kKeys ? (p->ctx + 3) / 4 * 4 : kKeys;
  e = fta_launch_after(evict_select_kernel, dim3(p->B * p->Hkv), kSelect, room * 4, st, 1, *p, room);
  if (e != cudaSuccess) return fta_cuda_fail(e);
  // Blocks until every SM has three (not every unit has rows to move): first the blocks of a cluster, which
  // share out a chunk's rows, then column slices down to 64 bytes, and to a 32-byte sector only where there
  // are fewer than two a SM.  A block moves some 20 GB/s: one unit of 13580 rows of 128 in 16 blocks (slices
  // of 32 bytes alone) took 25 us, in 32 (clusters of 8, 128 bytes) 15, in 128 (both) 6.
  const long long units = (long long)p->B * p->Hkv * 2;
  const int width = p->D / 8;
  int blocks = 1, slices = 1;
  while (units * blocks < 3 * kFtaSms && blocks < 8) blocks *= 2;
  while (units * blocks * slices < 4 * kFtaSms && blocks == 8 && width / slices > 4) slices *= 2;
  while (units * blocks * slices < 2 * kFtaSms && width / slices > 2) slices *= 2;
  e = fta_launch_after(evict_move_kernel, dim3(p->B * p->Hkv * blocks, 2, slices), kMove, 0, st, blocks, *p, width / slices, blocks);
  return e == cudaSuccess ? FTA_OK : fta_cuda_fail(e);
}
