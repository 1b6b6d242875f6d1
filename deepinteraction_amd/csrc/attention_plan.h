// How a launch of the attention kernels is cut into workgroups (host).
#pragma once
#include "attention.h"

namespace di {
namespace at {

struct Plan {
  int big;                               // rows: 0 = up to 16, 1 = up to 64, 2 = more; keys: tiles per wavefront
  int blocks, splits, range;
};

template <int TY>
int launch_fwd(const Args &a, const Plan &p, hipStream_t s);
template <int TY>
int launch_bwd(const Args &a, const Plan &gq, const Plan &gkv, hipStream_t s);

constexpr int padded(int D) { return D <= 16 ? 16 : D <= 32 ? 32 : D <= 64 ? 64 : 128; }
constexpr int row_tiles(int DP) { return DP <= 32 ? 4 : 2; }                       // MT of the large variant
constexpr int key_tiles(int TY, int DP) { return DP <= 32 ? 4 : (TY == DI_F32 && DP == 128 ? 1 : 2); }   // NT

}  // namespace at
}  // namespace di
