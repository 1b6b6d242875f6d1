// How a launch of the attention kernels is cut into workgroups (host).
#pragma once
#include "attention.h"

namespace di {
namespace at {

struct Plan {
  int big;                               // rows: 0 = up to 16, 1 = up to 64, 2 = more; keys: tiles per wavefront
  int blocks, splits, range;
  bool ragged;                           // workgroups with keys first
};

template <int TY>
int launch_fwd(const Args &a, const Plan &p, hipStream_t s);
template <int TY>
int launch_bwd(const Args &a, const Plan &gq, const Plan &gkv, hipStream_t s);

// (72 of 96 rather than of 128 dims, 2 x 1000 x 4000 x 8 heads: float32 305 + 430 + 573 -> 257 + 347 + 443 us, bf16 46 + 68 + 92 -> 45 + 52 + 87)
constexpr int padded(int D) { return D <= 16 ? 16 : D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }
constexpr int row_tiles(int DP) { return DP <= 32 ? 4 : 2; }                       // MT of the large variant
constexpr bool one_launch(int DP) { return DP <= 32; }                              // the backward's key-block kernel forms gq as well
// Key tiles per wavefront at the most.  Heads of 96 and 128: one, two wavefronts a SIMD (2048 x 8192 x 16 heads, bf16: 380 us; two tiles, whose
// sums leave room for one: 394).  Heads of 64: two (161 us; one: 189)
constexpr int key_tiles(int TY, int DP) { return DP == 16 ? 4 : DP == 32 ? (TY == DI_F32 ? 2 : 4) : DP == 64 ? 2 : 1; }
// With a (query, key) mask or dropout two at the most: their words and hashes take the registers of the second wavefront a SIMD (half precision, with four
// and with two: 2 x 200 x 32 400 x 8 heads of 16 and dropout 228 and 183 us with the join, 53 x 721 x 651 x 4 heads of 32 and a (query, key)
// mask 322 and 241)
constexpr int most_masked_key_tiles = 2;
constexpr int least_key_tiles(int DP) { return one_launch(DP) ? 2 : 1; }            // 16-bit products contract over 32 keys
// The joins: lanes across the head dim (a power of two), lanes per row - up to 64, the others on further ranges - and workgroups per problem.
struct JoinShape {
  int nd, group, blocks;
};
inline JoinShape join_shape(int D, int ranges, int rows) {
  JoinShape j;
  j.nd = (padded(D) == 96 ? 128 : padded(D)) / 4;
  j.group = j.nd;
  while (j.group < 64 && 4 * (j.group / j.nd) < ranges) j.group *= 2;
  const int per = 256 / j.group;
  j.blocks = (rows + per - 1) / per;
  return j;
}
constexpr int tile_rows(int TY, int DP) { return DP * (TY == DI_F32 ? 4 : 2) >= 512 || DP == 32 ? 32 : 64; }

}  // namespace at
}  // namespace di
