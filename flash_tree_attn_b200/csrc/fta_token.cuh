// Attention of one new token per sequence over the cache: split over the cache's length by the
// BALANCED plan (FtaBalanced), joined by a second kernel.
//
// Mathematics, per query head: s_r = scale * q.k_r (capped by c * tanh(s / c), plus slope * distance),
// out = sum_r 2^(s_r - m) v_r / sum_r 2^(s_r - m) with s in log2 units and a running m.
//
// What bounds it: every K and V row is read once per KV head, 4 * D bytes a row for 4 * D * G
// operations, 2 * G operations a byte: the cache stream (HBM) is the floor at any G <= 16.
//
// Layout.  A group's heads (8 or 16, padded) are the N side of mma.m16n8k16 and 16 cache rows its M
// side: S^T = K q^T, O^T = V^T P^T.  A contraction does not care for the order of its terms, so a lane
// takes 16 contiguous bytes of a K row as its part of two k-steps, and of V it takes 16 bytes of four
// rows, from which byte permutes make the pairs along the rows that the product wants.  Each warp copies
// and multiplies its own rows (16 of every 64-row tile) through a ring of its own, so no barrier but the
// warp's stands in the loop.  The warps meet once per piece, to join their (m, l, O).
//
// Measured: 64 ragged sequences of up to 8192 rows (32/8 heads of 128, pages of 64 rows, 1.1 GB of K and
// V): 179 us, 6.2 TB/s, 94 % of the measured copy rate.
#pragma once
#include "fta_common.cuh"

#define FTA_MAX_GROUP 256  // query heads per KV head

struct FtaTokenWs {  // byte offsets of the workspace's parts
  long long part_o, part_l, desc, lse2, scores, bytes;
};

// part_o [2 * grid][R][D] and part_l [2 * grid][R] as in FtaParams' BALANCED workspace (LSEs in log2
// units); desc [B * U] int2 {pieces, first group of blocks} per unit; with row weights also the log2
// LSE of every head [B * H] and every score [B * H][ctx, padded to whole 16 bytes] in log2 units.
__host__ __device__ __forceinline__ long long fta_token_pitch(int ctx) { return ((long long)ctx + 3) / 4 * 4; }
__host__ __device__ __forceinline__ FtaTokenWs fta_token_ws(int grid, int R, int D, int B, int U, int H, int ctx, bool weights) {
  FtaTokenWs w;
  w.part_o = 0;
  w.part_l = w.part_o + 2ll * grid * R * D * 4;
  w.desc = w.part_l + 2ll * grid * R * 4;
  w.lse2 = w.desc + (long long)B * U * 8;
  w.scores = (w.lse2 + (weights ? (long long)B * H * 4 : 0) + 15) / 16 * 16;
  w.bytes = w.scores + (weights ? (long long)B * H * fta_token_pitch(ctx) * 4 : 0);
  return w;
}

// first 64-row tile of a sequence that the window leaves in sight
__host__ __device__ __forceinline__ int fta_token_tile0(int L, int window) {
  return window > 0 && L > window ? (L - window) / FTA_TILE : 0;
}

cudaError_t fta_launch_token_d32(const FtaTokenParams&, const FtaGeom&, cudaStream_t, int, int*);
cudaError_t fta_launch_token_d64(const FtaTokenParams&, const FtaGeom&, cudaStream_t, int, int*);
cudaError_t fta_launch_token_d128(const FtaTokenParams&, const FtaGeom&, cudaStream_t, int, int*);
cudaError_t fta_launch_token_d256(const FtaTokenParams&, const FtaGeom&, cudaStream_t, int, int*);
