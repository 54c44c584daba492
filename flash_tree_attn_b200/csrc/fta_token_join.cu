// Joins the pieces of the one-token attention (fta_token.cuh), finishes the rows of empty sequences
// and adds the softmax weights of the group's heads to row_weights.
//
// out = sum_i 2^(l_i - M) o_i / sum_i 2^(l_i - M) over the pieces' log2 LSEs l_i.  Row weights:
// w_r += sum_h 2^(s_hr - LSE_h) from the scores stage 1 kept, so K is not read a second time
// (4 G bytes a row instead of 2 D).
//
// grid = (B * Hkv, max(shares, chunks of the cache's length)).  The group's heads are dealt out to the first
// `shares` blocks of a KV head, and the pieces of a head to the block's warps where it has fewer heads
// than warps: a few long units have up to a hundred pieces each.  With row weights every block works
// all heads' LSEs out for itself and has a chunk of rows.
#include "fta_token.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// eviction orders weights by their bits, so a row that gains nothing keeps its own, subnormal ones too, which
// the compiler's addition takes for zero (--use_fast_math)
__device__ __forceinline__ float add_kept(float a, float b) {
  float y;
  asm("add.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

__global__ void __launch_bounds__(kThreads, 3) token_join_kernel(const FtaTokenParams p, const FtaGeom g, const int shares, const int chunk_rows) {
  __shared__ float s_lse[FTA_MAX_GROUP];
  __shared__ __align__(16) float s_o[kWarps][128];
  __shared__ float s_top[kWarps], s_sum[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x / p.Hkv, kvh = blockIdx.x - b * p.Hkv;
  const int G = p.H / p.Hkv, lanes = g.lanes > 0 ? g.lanes : 1;
  const bool weights = p.row_weights != nullptr;
  const FtaTokenWs ws = fta_token_ws(g.grid, g.R, p.D, p.B, g.U, p.H, p.ctx, weights);
  const uint8_t* wsb = reinterpret_cast<const uint8_t*>(p.workspace);
  const float* part_o = reinterpret_cast<const float*>(wsb + ws.part_o);
  const float* part_l = reinterpret_cast<const float*>(wsb + ws.part_l);
  const int2* desc = reinterpret_cast<const int2*>(wsb + ws.desc);
  const float* lse2 = reinterpret_cast<const float*>(wsb + ws.lse2);

  fta_after_previous();

  const int L = fta_load_len(p.kv_seq_len, p.len_is_i64, b, p.ctx);
  const int row0 = blockIdx.y * chunk_rows;
  // {pieces, first group of blocks} of head hh's unit
  auto pieces_of = [&](int hh) {
    const int2 d = desc[(long long)b * g.U + kvh * g.n_gt + hh / g.R];  // asked for together with the length, which
    return L > 0 ? d : make_int2(0, 0);                                 // says whether it was written
  };
  // row of piece i of head hh among the partial rows
  auto slot = [&](int hh, int first, int i) {
    const int lane_of = g.lanes > 1 ? hh / g.R : 0;
    return ((long long)2 * ((first + i) * lanes + lane_of) + (i == 0 ? 1 : 0)) * g.R + hh % g.R;
  };

  if ((int)blockIdx.y < shares) {
    const int heads = (G - 1 - (int)blockIdx.y) / shares + 1, columns = p.D > 128 ? 2 : 1;  // blockIdx.y < shares <= G
    const int tasks = heads * columns;
    const int team = tasks > 4 ? 1 : tasks > 2 ? 2 : tasks > 1 ? 4 : 8;  // warps per task
    for (int t0 = 0; t0 < tasks; t0 += kWarps / team) {
      const int t = t0 + warp / team, member = warp % team;
      const int hh = blockIdx.y + shares * (t / columns), h = kvh * G + hh, c4 = (t % columns) * 128 + lane * 4;
      const bool live = t < tasks, inside = c4 < p.D;
      const int2 d = live ? pieces_of(hh) : make_int2(1, 0);
      float top = -INFINITY, sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      if (d.x > 1) {
        for (int i0 = member; i0 < d.x; i0 += 32 * team) {  // lane j has the LSE of piece i0 + team j
          const int i = i0 + team * lane, count = min(32, fta_cdiv(d.x - i0, team));
          const float l = i < d.x ? part_l[slot(hh, d.y, i)] : -INFINITY;
          const float now = fmaxf(top, warp_max(l)), base = now == -INFINITY ? 0.f : now;
          const float keep = fta_exp2(top - base), w = fta_exp2(l - base);  // NaN stays in sight in w
          acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
          sum = sum * keep + warp_sum(w);
          top = now;
          for (int j0 = 0; j0 < count; j0 += 8) {  // eight pieces' loads go out together
            float4 x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
              x[u] = j0 + u < count && inside ? *reinterpret_cast<const float4*>(part_o + slot(hh, d.y, i0 + team * (j0 + u)) * p.D + c4)
                                              : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const float f = __shfl_sync(0xffffffffu, w, (j0 + u) & 31);
              acc.x += f * x[u].x; acc.y += f * x[u].y; acc.z += f * x[u].z; acc.w += f * x[u].w;
            }
          }
        }
      }
      if (team > 1) {
        *reinterpret_cast<float4*>(&s_o[warp][lane * 4]) = acc;
        if (lane == 0) { s_top[warp] = top; s_sum[warp] = sum; }
        __syncthreads();
        if (member == 0) {
          const float mine = lane < team ? s_top[warp + lane] : -INFINITY;
          top = warp_max(mine);
          const float base = top == -INFINITY ? 0.f : top;
          sum = 0.f;
          acc = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int m = 0; m < team; ++m) {
            const float f = fta_exp2(s_top[warp + m] - base);
            const float4 x = *reinterpret_cast<const float4*>(&s_o[warp + m][lane * 4]);
            acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
            sum += f * s_sum[warp + m];
          }
        }
        __syncthreads();
      }
      if (live && member == 0 && d.x != 1) {  // 1: stage 1 wrote the row itself; 0: no rows, zeros
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        if (inside)
          fta_store4(p.out, p.dtype, b * p.o_sb + h * p.o_sh + c4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
        if (c4 == 0 && p.lse) p.lse[b * p.l_sb + h] = sum == 0.f ? -INFINITY : (top + fta_log2(sum)) * FTA_LN2;
      }
    }
  }
  if (!weights || row0 >= L) return;

  for (int hh = warp; hh < G; hh += kWarps) {
    const int2 d = pieces_of(hh);
    float total = -INFINITY;
    if (d.x == 1) {
      total = lse2[(long long)b * p.H + kvh * G + hh];
    } else {
      float l[4], top = -INFINITY, sum = 0.f;
      for (int i0 = 0; i0 < d.x; i0 += 128) {
#pragma unroll
        for (int u = 0; u < 4; ++u) l[u] = i0 + 32 * u + lane < d.x ? part_l[slot(hh, d.y, i0 + 32 * u + lane)] : -INFINITY;
        const float now = fmaxf(top, warp_max(fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])))), base = now == -INFINITY ? 0.f : now;
        sum = sum * fta_exp2(top - base) + warp_sum(fta_exp2(l[0] - base) + fta_exp2(l[1] - base) + fta_exp2(l[2] - base) + fta_exp2(l[3] - base));
        top = now;
      }
      total = sum == 0.f ? -INFINITY : top + fta_log2(sum);
    }
    if (lane == 0) s_lse[hh] = total;
  }
  __syncthreads();
  // A thread has four consecutive rows and asks for eight heads' scores of them together: the loop waits
  // for memory and for nothing else.
  const long long pitch = fta_token_pitch(p.ctx);
  const float* scores = reinterpret_cast<const float*>(wsb + ws.scores) + ((long long)b * p.H + kvh * G) * pitch;
  float* out = p.row_weights + b * p.rw_sb + kvh * p.rw_sh;
  const int first = p.window > 0 ? max(0, L - p.window) : 0;
  const int end = min(L, row0 + chunk_rows);
#pragma unroll 1
  for (int row = row0 + 4 * (int)threadIdx.x; row < end; row += 4 * kThreads) {
    if (row + 3 < first) continue;
    float old[4], w[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e) old[e] = row + e >= first && row + e < L ? out[row + e] : 0.f;
    for (int h0 = 0; h0 < G; h0 += 8) {
      float4 x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (h0 + u < G) x[u] = __ldcs(reinterpret_cast<const float4*>(scores + (h0 + u) * pitch + row));
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float total = h0 + u < G ? s_lse[h0 + u] : -INFINITY;
        if (total == -INFINITY) continue;
        w[0] += fta_exp2(x[u].x - total);
        w[1] += fta_exp2(x[u].y - total);
        w[2] += fta_exp2(x[u].z - total);
        w[3] += fta_exp2(x[u].w - total);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (row + e >= first && row + e < L) out[row + e] = add_kept(old[e], w[e]);
  }
}

template <typename F>
int token_variant(const FtaTokenParams& p, F&& f) {
  switch (p.D) {
    case 32: return f(fta_launch_token_d32);
    case 64: return f(fta_launch_token_d64);
    case 128: return f(fta_launch_token_d128);
  }
  return f(fta_launch_token_d256);
}

bool aligned16(const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }

int check_sizes(const FtaTokenParams* p) {
  if (!p || p->B <= 0 || p->H <= 0 || p->Hkv <= 0 || p->ctx < 0 || p->H % p->Hkv != 0) return FTA_E_BADARG;
  if (p->D != 32 && p->D != 64 && p->D != 128 && p->D != 256) return FTA_E_BADARG;
  if (p->dtype != FTA_DTYPE_F16 && p->dtype != FTA_DTYPE_BF16) return FTA_E_BADARG;
  if (p->grid_override < 0) return FTA_E_BADARG;
  if (p->B > FTA_MAX_BATCH || p->H / p->Hkv > FTA_MAX_GROUP || p->ctx > FTA_MAX_ROWS) return FTA_E_UNSUPPORTED;
  // the plan counts all sequences' 64-row tiles, and a few more each, in 32 bits
  const int rows = p->window > 0 && p->window < p->ctx ? p->window + FTA_TILE : p->ctx;
  if ((long long)p->B * (fta_cdiv(rows, FTA_TILE) + 8) > 0x7fffffffLL) return FTA_E_UNSUPPORTED;
  return FTA_OK;
}

int check(const FtaTokenParams* p) {
  if (int rc = check_sizes(p)) return rc;
  if (!p->q || !p->kv_seq_len || !p->out || (p->ctx > 0 && (!p->k_cache || !p->v_cache))) return FTA_E_BADARG;
  if (!aligned16(p->q) || !aligned16(p->k_cache) || !aligned16(p->v_cache) || !aligned16(p->out)) return FTA_E_BADARG;
  for (int64_t s : {p->q_sb, p->q_sh, p->k_sb, p->k_sh, p->k_st, p->v_sb, p->v_sh, p->v_st})
    if (s % 8 != 0) return FTA_E_BADARG;
  if (p->o_sb % 4 != 0 || p->o_sh % 4 != 0) return FTA_E_BADARG;
  if (!(p->softcap >= 0.f) || p->window < 0) return FTA_E_BADARG;
  if (p->block_table) {
    if (p->page_size < FTA_TILE || p->page_size % FTA_TILE != 0 || p->n_pages < 1 || p->bt_sb < 0) return FTA_E_BADARG;
    if ((long long)p->bt_sb * p->page_size < p->ctx && p->B > 1) return FTA_E_BADARG;
  }
  if (!aligned16(p->workspace)) return FTA_E_WORKSPACE;
  return FTA_OK;
}

// [device][dtype][head_dim][rows][KB of the prefix table] -> resident blocks per SM, 0: not asked yet
int g_occ[16][2][4][2][34];
int g_sms[16];

int geometry(const FtaTokenParams& p, FtaGeom& g) {
  const int G = p.H / p.Hkv;
  // 16 padded heads cost twice the products and accumulators of 8: only where a group has more than 8,
  // and not at head_dim 256, whose accumulators would spill; there two blocks share the rows through L2
  g.R = G > 8 && p.D < 256 ? 16 : 8;
  g.qpt = 1; g.n_qt = 1;
  g.hpt = g.R;
  g.n_gt = fta_cdiv(G, g.R);
  g.mtiles = g.n_gt;
  g.U = p.Hkv * g.n_gt;
  g.n_tree = 0;
  g.min_per = 1;
  g.fixed_max_splits = 0; g.family = 0; g.cs = 1;
  g.pad = 4;  // as the warp-MMA family; 0 to 4 lie within 2 % of each other
  g.grid = p.grid_override;
  if (p.grid_override == 0) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return fta_cuda_fail(e);
    int& sms = g_sms[dev & 15];
    if (sms == 0 && (e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return fta_cuda_fail(e);
    const int d = p.D == 32 ? 0 : p.D == 64 ? 1 : p.D == 128 ? 2 : 3;
    int& occ = g_occ[dev & 15][p.dtype][d][g.R == 16][((p.B + 1) * 4) / 1024];
    if (occ == 0) {
      int n = 0;
      e = (cudaError_t)token_variant(p, [&](auto launch) { return (int)launch(p, g, 0, 1, &n); });
      if (e != cudaSuccess) return fta_cuda_fail(e);
      if (n < 1) return FTA_E_UNSUPPORTED;
      occ = n;
    }
    g.grid = sms * occ;
  }
  g.lanes = g.mtiles > 1 && g.grid >= g.mtiles ? g.mtiles : 1;
  // Short caches: one launch, a cluster of blocks per unit that joins without a second kernel.  It shares
  // out each unit's tiles evenly but not those of different lengths, so no block may get more than 8 tiles
  // (16 of a single sequence, 8192 rows in clusters of 8), and all clusters are resident at once.  The rule goes
  // by the cache's capacity or the window: lengths are on the device, so a short sequence in a large cache takes
  // the BALANCED plan.  On the GPU, clusters against the BALANCED plan, 32/8 heads of 128: one sequence of 1000
  // rows 4.7 and 8.3 us, of 4000 8.1 and 11.5; 8 sequences of 2000 rows 14.5 and 18.7.  Without the limit one
  // sequence of 16000 rows took 22.1 and 22.9: little was left of the gain.
  if (p.grid_override == 0 && !p.row_weights && p.B <= 4096) {
    const int rows = p.window > 0 && p.window < p.ctx ? p.window + FTA_TILE - 1 : p.ctx;
    const int tiles = rows > 0 ? fta_cdiv(rows, FTA_TILE) : 1;
    const int units = p.B * g.U;
    for (int c = 8; c >= 1; c /= 2) {
      if (units > g.grid / c || tiles > (p.B == 1 ? 16 : 8) * c || (c > 1 && tiles <= c / 2)) continue;
      g.family = 1;
      g.cs = c;
      g.grid = units * c;
      break;
    }
  }
  return FTA_OK;
}

long long workspace_of(const FtaTokenParams& p, const FtaGeom& g) {
  return g.family == 1 ? 0 : fta_token_ws(g.grid, g.R, p.D, p.B, g.U, p.H, p.ctx, p.row_weights != nullptr).bytes;
}

}  // namespace

extern "C" int64_t fta_decode_token_workspace_bytes(const FtaTokenParams* p) {
  if (int rc = check_sizes(p)) return -rc;
  FtaGeom g;
  if (int rc = geometry(*p, g)) return -rc;
  return workspace_of(*p, g);
}

extern "C" int fta_decode_token(const FtaTokenParams* p, void* stream) {
  if (int rc = check(p)) return rc;
  FtaGeom g;
  if (int rc = geometry(*p, g)) return rc;
  const bool weights = p->row_weights != nullptr;
  const long long need = workspace_of(*p, g);
  if (need > 0 && (!p->workspace || p->workspace_bytes < need)) return FTA_E_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = (cudaError_t)token_variant(*p, [&](auto launch) { return (int)launch(*p, g, st, 0, nullptr); });
  if (e != cudaSuccess) return fta_cuda_fail(e);
  if (g.family == 1) return FTA_OK;
  int chunk = 4 * kThreads;
  while (weights && fta_cdiv(p->ctx, chunk) > 65535) chunk *= 2;  // a grid's second dimension ends there
  const int chunks = weights ? fta_cdiv(p->ctx, chunk) : 0;
  // a block per head where there are few KV heads: then a unit has many pieces
  const int shares = p->B * p->Hkv < kFtaSms ? p->H / p->Hkv : 1;
  const dim3 grid(p->B * p->Hkv, shares > chunks ? shares : chunks);
  e = fta_launch_after(token_join_kernel, grid, kThreads, 0, st, 1, *p, g, shares, chunk);
  return e == cudaSuccess ? FTA_OK : fta_cuda_fail(e);
}
