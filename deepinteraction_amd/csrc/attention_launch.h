// Dispatch of the attention kernels of one element type by head dim and variant.
#pragma once
#include "attention_bwd.h"
#include "attention_plan.h"

namespace di {
namespace at {

static bool needs_full(const Args &a) { return a.kmask != nullptr || a.allowed != nullptr || a.drop != 0; }

template <class K>
static int go(K kernel, LdsRaised &raised, int lds, long long grid, const Args &a, hipStream_t s, const char *name) {
  if (grid <= 0) return DI_OK;
  if (int rc = ensure_lds(raised, (const void *)kernel, lds)) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), lds, s, a);
  return check_launch(name);
}

template <int TY, bool STATS>
static int join(const Args &args, hipStream_t s) {
  Args a = args;
  const JoinShape j = join_shape(a.D, a.splits, a.G * a.L);
  a.by_unit = div_by(j.blocks);
  hipLaunchKernelGGL((attention_join_kernel<TY, STATS>), dim3((unsigned)(a.B * a.Hk * j.blocks)), dim3(256), 0, s, a, j.nd, j.group);
  return check_launch("attention_join");
}

template <int TY, int DP, int MT, int WQ>
static int fwd(const Args &a, hipStream_t s) {
  static LdsRaised plain, full;
  const long long grid = (long long)a.B * a.splits * a.Hk * a.blocks;
  constexpr int lds = FwdCfg<TY, DP, MT, WQ>::LDS;
  return needs_full(a) ? go(attention_fwd_kernel<TY, DP, MT, WQ, true>, full, lds, grid, a, s, "attention_fwd")
                       : go(attention_fwd_kernel<TY, DP, MT, WQ, false>, plain, lds, grid, a, s, "attention_fwd");
}
template <int TY, int DP, int MT, int WQ>
static int gq(const Args &a, hipStream_t s) {
  static LdsRaised plain, full;
  const long long grid = (long long)a.B * a.splits * a.Hk * a.blocks;
  constexpr int lds = GqCfg<TY, DP, MT, WQ>::LDS;
  if constexpr (DP >= 96 && MT > 1 && TY != DI_F32) {                          // the plan: 64 rows with masks and dropout
    return go(attention_gq_kernel<TY, DP, MT, WQ, false>, plain, lds, grid, a, s, "attention_gq");
  } else {
    return needs_full(a) ? go(attention_gq_kernel<TY, DP, MT, WQ, true>, full, lds, grid, a, s, "attention_gq")
                         : go(attention_gq_kernel<TY, DP, MT, WQ, false>, plain, lds, grid, a, s, "attention_gq");
  }
}
template <int TY, int DP, int NT>
static int gkv(const Args &a, hipStream_t s) {
  static LdsRaised plain, full;
  const long long grid = (long long)a.B * a.splits * a.Hk * a.blocks;
  constexpr bool GQ = one_launch(DP);
  using C = GkvCfg<TY, DP, NT, GQ>;
  static_assert(C::BR == tile_rows(TY, DP) && C::LDS % 16 == 0, "the plan's tiles; the mask's words");
  if constexpr (NT <= most_masked_key_tiles) {
    if (a.allowed != nullptr || a.drop != 0 || a.S <= kFew) return go(attention_gkv_kernel<TY, DP, NT, GQ, true>, full, C::LDS + C::MASK + C::DROP, grid, a, s, "attention_gkv");
  }
  return go(attention_gkv_kernel<TY, DP, NT, GQ, false>, plain, C::LDS, grid, a, s, "attention_gkv");
}

// walk: the keys per range (row blocks) or per block (key blocks)
static void take(Args &a, const Plan &p, int walk, int inner) {
  a.blocks = p.blocks;
  a.splits = p.splits;
  a.range = p.range;
  const int unit = a.blocks * a.Hk, units = a.B * a.splits;
  a.even = units / 8 * 8 * unit;
  a.by_unit = div_by(unit);
  a.by_blocks = div_by(a.blocks);
  a.by_hk = div_by(a.Hk);
  a.by_splits = div_by(a.splits);
  a.by_L = div_by(a.L);
  a.ragged = p.ragged;
  a.by_walk = div_by(walk);
  a.by_inner = div_by(inner);
}

template <int TY>
int launch_fwd(const Args &args, const Plan &p, hipStream_t s) {
  Args a = args;
  take(a, p, p.range, p.blocks * a.Hk);
  int rc;
#define DI_AT_FWD(DP) \
  rc = p.big == 0 ? fwd<TY, DP, 1, 1>(a, s) : p.big == 1 ? fwd<TY, DP, 1, 4>(a, s) : fwd<TY, DP, row_tiles(DP), 4>(a, s)
  switch (padded(a.D)) {
    case 16: DI_AT_FWD(16); break;
    case 32: DI_AT_FWD(32); break;
    case 64: DI_AT_FWD(64); break;
    case 96: DI_AT_FWD(96); break;
    default: DI_AT_FWD(128); break;
  }
#undef DI_AT_FWD
  if (rc != DI_OK || p.splits == 1) return rc;
  return join<TY, true>(a, s);
}

template <int TY>
int launch_bwd(const Args &args, const Plan &pq, const Plan &pk, hipStream_t s) {
  Args a = args;
  int rc = DI_OK;
  if (!one_launch(padded(a.D))) {
    take(a, pq, pq.range, pq.blocks * a.Hk);
#define DI_AT_GQ(DP) \
  rc = pq.big == 0 ? gq<TY, DP, 1, 1>(a, s) : pq.big == 1 ? gq<TY, DP, 1, 4>(a, s) : gq<TY, DP, row_tiles(DP), 4>(a, s)
    if (a.L > 0) {
      if (padded(a.D) == 64) DI_AT_GQ(64);
      else if (padded(a.D) == 96) DI_AT_GQ(96);
      else DI_AT_GQ(128);
    }
#undef DI_AT_GQ
    if (rc != DI_OK) return rc;
    if (a.L > 0 && pq.splits > 1 && (rc = join<TY, false>(a, s)) != DI_OK) return rc;
    if (a.S == 0) return DI_OK;
  }
  take(a, pk, 64 * pk.big, pk.splits * a.Hk);
#define DI_AT_GKV(DP)                                                                                                      \
  do {                                                                                                                     \
    constexpr int most = key_tiles(TY, DP), least = least_key_tiles(DP);                                                   \
    rc = pk.big >= 4 && most >= 4 ? gkv<TY, DP, most >= 4 ? 4 : least>(a, s)                                               \
         : pk.big >= 2 && most >= 2 ? gkv<TY, DP, most >= 2 ? 2 : least>(a, s)                                             \
                                    : gkv<TY, DP, least>(a, s);                                                            \
  } while (0)
  switch (padded(a.D)) {
    case 16: DI_AT_GKV(16); break;
    case 32: DI_AT_GKV(32); break;
    case 64: DI_AT_GKV(64); break;
    case 96: DI_AT_GKV(96); break;
    default: DI_AT_GKV(128); break;
  }
#undef DI_AT_GKV
  if (rc != DI_OK) return rc;
  if (one_launch(padded(a.D)) && pk.blocks > 1 && a.L > 0) {
    Args j = a;                                                 // the join's ranges are the key blocks
    j.splits = pk.blocks;
    j.range = 64 * pk.big;
    if ((rc = join<TY, false>(j, s)) != DI_OK) return rc;
  }
  if (pk.splits == 1 || a.S == 0) return DI_OK;
  const long long n = (long long)a.B * a.Hk * a.S * (a.D / 4);
  hipLaunchKernelGGL((attention_gkv_join_kernel<TY>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a);
  return check_launch("attention_gkv_join");
}

}  // namespace at
}  // namespace di
