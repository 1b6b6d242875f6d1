// Backward of the attention to another sequence (attention_fwd.h).  With p_j = exp2(scale2 q . k_j - lse), dp_j = go . v_j,
// delta = go . o and ds_j = p_j (dp_j - delta):
//
//     gq = scale sum_j ds_j k_j        gk_j = scale sum_rows ds_j q        gv_j = sum_rows p_j go
//
// Two launches, neither with atomics, both deterministic: `gq` keeps a block of rows in registers and walks over the keys (the
// forward's structure; it also writes delta), `gk, gv` keeps a block of keys and walks over the rows.  Both form the scores again:
// 14 D instead of 10 D operations a pair, but no partial result of the long side ever leaves the chip.
//   gq:      S^T = K Q^T, dP^T = V go^T (16 keys x 16 rows), gq^T += K^T dS^T
//   gk, gv:  S = Q K^T, dP = go V^T (16 rows x 16 keys), gv^T += go^T P, gk^T += Q^T dS
// Where there are few blocks, the walked side is split over workgroups and their float32 sums are added in a fixed order.
// Heads of up to 32 dims: ONE launch.  The key-block kernel forms gq as well - every wavefront from its own keys, its score gradients
// transposed through LDS, the four shares added per tile of rows, the key blocks' sums joined by the forward's second launch.  The
// scores are formed once, and rows of few dims make the key blocks' sums small (rows x D floats per 128 - 256 keys); wide heads would
// write more sums than the second pass over the keys costs.
//
// What bounds them, and what they measured (shares of the SIMDs' cycles from the counters of the final build):
//   heads of 128 (2048 x 8192 x 16, bf16): gq 256 - 269 us = 770 - 805 TFLOP/s, gk and gv 356 - 375 us = 730 - 770: matrix cores 38 %, vector
//     unit 32; gq has one wavefront a SIMD, gk and gv two that hold 16 keys each, so every fragment of Q and go from LDS feeds one product
//     (LDS works in 53 % of the cycles) and the wavefronts wait 42 % of theirs for a unit to take their next instruction
//   heads of 64, four to a key head (4 x 511 x 4100, 2733, 1366, 0, bf16): gq 47 us, gk and gv 79: 264 workgroups for 256 CUs, one
//     wavefront a SIMD (1.15) - its own chain of product, exponential, product is the time of a tile
//   heads of 16, one launch: 200 x 32 400 x 8, float32: 102 us, matrix cores 64 %, vector unit 24; half precision, 2 samples: 67 us, vector
//     unit 62 %, and 1200 x 60 x 112: 78 us, 56 % (ten instructions and an exponential a pair)
// Attention dropout, p = 0.1 (forward and backward): the hashes of a pair, formed in both directions - float32 200 x 32 400: 52 + 101 -> 62 +
// 130 us; half precision, 2 samples: 41 + 71 -> 70 + 138; 1200 x 60 x 112: 31 + 68 -> 49 + 111.
// Spilled registers: masked gk and gv of 16-bit heads of 64 (19, 48 bytes of scratch, at the bound of two wavefronts a SIMD; 1024 x 4096 x 8:
// the whole backward 97 us with a (query, key) mask, 68 without) and float32 masked gq of 128 dims (4 of its accumulation registers).
// Not taken: the products over a chunk's rows left for the next chunk, to hide behind its exponentials - the registers that this takes
// cost the second wavefront of the SIMD (4 x 511 x .. of 64: 79 -> 110 us; heads of 128: 410 -> 433).
#pragma once
#include "attention_fwd.h"

namespace di {
namespace at {

template <int TY, int DP, int MT, int WQ>
struct GqCfg {
  using M = Mm<TY, DP>;
  static constexpr int WK = 4 / WQ;
  static constexpr int CPT = WQ == 1 ? 1 : 64 / M::CH;
  static constexpr int TILE = WK * CPT * M::CH;
  static constexpr int V_AT = TILE * M::TRS, BIAS_AT = V_AT + TILE * M::ROWS;
  static constexpr int JOIN = WQ == 1 ? 4 * 16 * DP * 4 : 0;
  static constexpr int LDS = BIAS_AT + TILE * 4 > JOIN ? BIAS_AT + TILE * 4 : JOIN;
  static constexpr int ROWS_PER_BLOCK = 16 * MT * WQ;
  static constexpr int NP = (TILE * M::PPR + 255) / 256;
};

template <int TY, int DP, int MT, int WQ, bool FULL>
__global__ __launch_bounds__(256) void attention_gq_kernel(Args a) {
  using C = GqCfg<TY, DP, MT, WQ>;
  using M = Mm<TY, DP>;
  extern __shared__ __align__(16) char lds[];
  float *bias = reinterpret_cast<float *>(lds + C::BIAS_AT);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
  const Where at = where<false>(a);
  const int wq = WQ == 1 ? 0 : (wave + at.sp + at.hk + at.b) % WQ, wk = wave / WQ;
  const int rows = a.G * a.L, ntile = (rows + 15) / 16;
  const int nkeys = keys_of(a, at.b), k0 = at.sp * a.range, k1 = min(k0 + a.range, nkeys);
  const bool few = a.S <= kFew;
  const char *kb = a.k + at.b * a.k_bs + (long long)at.hk * a.D * M::SZ, *vb = a.v + at.b * a.v_bs + (long long)at.hk * a.D * M::SZ;
  const unsigned char *km = !FULL || a.kmask == nullptr ? nullptr : a.kmask + at.b * a.kmask_bs;
  const long long row_id = ((long long)at.b * a.Hk + at.hk) * rows;

  typename M::RF qf[MT][M::NK], gf[MT][M::NK];
  f4 acc[MT][M::ND];
  float lse[MT], delta[MT];
  int row[MT], query[MT];
  unsigned drow[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int tile = (at.blk * MT + t) * WQ + wq;
    row[t] = tile < ntile ? 16 * tile + i : rows;
    const bool ok = row[t] < rows;
    const int r = min(row[t], rows - 1), head = a.G == 1 ? 0 : (int)a.by_L.of(r);
    query[t] = r - head * a.L;
    const long long col = (long long)(at.hk * a.G + head) * a.D * M::SZ;
    const char *qp = a.q + at.b * a.q_bs + query[t] * a.q_rs + col, *gp = a.go + at.b * a.go_bs + query[t] * a.go_rs + col;
    const char *op = a.o + ((long long)at.b * a.L + query[t]) * a.Hk * a.G * a.D * M::SZ + col;
    float d = 0.f;
#pragma unroll
    for (int kk = 0; kk < M::NK; ++kk) {
      qf[t][kk] = M::row_frag_of(qp, kk, g, a.D, ok);
      gf[t][kk] = M::row_frag_of(gp, kk, g, a.D, ok);
      d += M::widen_dot(gf[t][kk], M::row_frag_of(op, kk, g, a.D, ok));
    }
    d += __shfl_xor(d, 16);
    d += __shfl_xor(d, 32);
    const float e = ok ? a.lse[row_id + r] : INFINITY;
    lse[t] = e == -INFINITY ? INFINITY : e;                     // an empty row: every probability 0, and no gradient whatever it holds
    if (few && ok && one_key(a, at.b, query[t], nkeys)) lse[t] = INFINITY;
    if (e == -INFINITY) d = 0.f;
    delta[t] = d;
    if (ok && at.sp == 0 && wk == 0 && g == 0) a.delta[row_id + row[t]] = d;
#pragma unroll
    for (int j = 0; j < M::ND; ++j) acc[t][j] = f4{0.f, 0.f, 0.f, 0.f};
    drow[t] = FULL && a.drop ? drop_row(seed_of(a), row_id + r) : 0;
  }
  if (a.splits > 1 && k0 >= k1) return;

  auto tile = [&](auto edge, int t0) {                          // one tile of keys; EDGE: keys are tested
    constexpr bool EDGE = decltype(edge)::value;
#pragma unroll
    for (int c = 0; c < C::CPT; ++c) {
      const int kc = (wk * C::CPT + c) * M::CH;
      if (EDGE && t0 + kc >= k1) break;
      unsigned may[MT][M::NT];                                  // in flight behind the products
      if (FULL && a.allowed != nullptr) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int u = 0; u < M::NT; ++u)
            may[t][u] = look<EDGE>(a.allowed + at.b * a.allowed_bs + query[t] * a.allowed_rs, t0 + kc + 16 * u + 4 * g, a.S);
      }
      f4 s[MT][M::NT], dp[MT][M::NT];
#pragma unroll
      for (int u = 0; u < M::NT; ++u) {
#pragma unroll
        for (int t = 0; t < MT; ++t) s[t][u] = dp[t][u] = f4{0.f, 0.f, 0.f, 0.f};
        typename M::RF kf[M::NK], vf[M::NK];                    // the tile's fragments before its first product
#pragma unroll
        for (int kk = 0; kk < M::NK; ++kk) {
          kf[kk] = M::row_frag_x(lds + (kc + 16 * u + i) * M::TRS, kk, g, i);
          vf[kk] = M::row_frag(lds + C::V_AT + (kc + 16 * u + i) * M::ROWS, kk, g);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < M::NK; ++kk)
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            s[t][u] = M::dot(kf[kk], qf[t][kk], s[t][u]);
            dp[t][u] = M::dot(vf[kk], gf[t][kk], dp[t][u]);
          }
        if (EDGE) {
          const f4 bb = *reinterpret_cast<const f4 *>(bias + kc + 16 * u + 4 * g);
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[t][u][r] = bb[r] == 0.f ? s[t][u][r] : -INFINITY;
        }
        if (FULL && a.allowed != nullptr) {
#pragma unroll
          for (int t = 0; t < MT; ++t) exclude(moved<EDGE>(may[t][u], t0 + kc + 16 * u + 4 * g, a.S), s[t][u]);
        }
      }
      typename M::TF kt[M::ND];                                 // in flight behind the exponentials
#pragma unroll
      for (int d = 0; d < M::ND; ++d) kt[d] = M::tr_frag(lds, M::TRS, kc, d, i, g);
      __builtin_amdgcn_sched_barrier(0);
      typename M::PF df[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        f4 ds[M::NT];
#pragma unroll
        for (int u = 0; u < M::NT; ++u) {
          if (FULL && a.drop) {
            const unsigned k4 = (unsigned)(t0 + kc + 16 * u + 4 * g) >> 2;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const unsigned x = drop_pair(drow[t], k4, h);
              dp[t][u][2 * h] = (x & 0xffffu) >= a.drop ? dp[t][u][2 * h] * a.keep_scale : 0.f;
              dp[t][u][2 * h + 1] = (x >> 16) >= a.drop ? dp[t][u][2 * h + 1] * a.keep_scale : 0.f;
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r)
            ds[u][r] = __builtin_amdgcn_exp2f(fmaf(s[t][u][r], a.scale2, -lse[t])) * (dp[t][u][r] - delta[t]);
          M::pack(df[t], u, ds[u]);
        }
      }
#pragma unroll
      for (int d = 0; d < M::ND; ++d)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t][d] = M::acc(kt[d], df[t], acc[t][d]);
    }
  };

  KeyStage<C> st;
  st.init(a);
  if (k0 < k1) st.fetch(a, kb, vb, km, k0, k1);
  auto step = [&](auto edge, int t0) {
    __syncthreads();
    st.template commit<true, false>(lds, C::V_AT, km != nullptr);
    if (decltype(edge)::value && threadIdx.x < C::TILE) {
      const int s = t0 + threadIdx.x;
      bias[threadIdx.x] = s < k1 && (km == nullptr || km[s] != 0) ? 0.f : -INFINITY;
    }
    __syncthreads();
    if (t0 + C::TILE < k1) st.fetch(a, kb, vb, km, t0 + C::TILE, k1);
    tile(edge, t0);
  };
  int t0 = k0;
  if (km == nullptr)
    for (; t0 + C::TILE <= k1; t0 += C::TILE) step(std::false_type(), t0);
  for (; t0 < k1; t0 += C::TILE) step(std::true_type(), t0);

  if (FULL) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int d = 0; d < M::ND; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[t][d][r] = lse[t] == INFINITY ? 0.f : acc[t][d][r];
  }
  if constexpr (WQ == 1) {                                      // add the four wavefronts (MT = 1)
    float *j = reinterpret_cast<float *>(lds);
    __syncthreads();
#pragma unroll
    for (int d = 0; d < M::ND; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) j[(wave * 16 + i) * DP + 16 * d + 4 * g + r] = acc[0][d][r];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int d = 0; d < M::ND; ++d)
#pragma unroll
      for (int w = 1; w < 4; ++w)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[0][d][r] += j[(w * 16 + i) * DP + 16 * d + 4 * g + r];
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    if (row[t] >= rows) continue;
    if (a.splits > 1) {
      float *p = a.part + ((long long)at.sp * a.B * a.Hk * rows + row_id + row[t]) * a.D;
#pragma unroll
      for (int d = 0; d < M::ND; ++d)
        if (16 * d + 4 * g < a.D) *reinterpret_cast<f4 *>(p + 16 * d + 4 * g) = acc[t][d];
    } else {
      const int head = a.G == 1 ? 0 : (int)a.by_L.of(row[t]);
      char *p = a.gq + (((long long)at.b * a.L + query[t]) * a.Hk * a.G + at.hk * a.G + head) * a.D * M::SZ;
#pragma unroll
      for (int d = 0; d < M::ND; ++d)
        if (16 * d + 4 * g < a.D) M::store4(p + (16 * d + 4 * g) * M::SZ, acc[t][d] * a.scale);
    }
  }
}

// GQ: the launch forms gq as well (narrow heads)
template <int TY, int DP, int NT, bool GQ>
struct GkvCfg {
  using M = Mm<TY, DP>;
  static constexpr int BR = DP * M::SZ >= 512 || (GQ && DP > 16) ? 32 : 64;        // rows per tile
  static constexpr int KEYS = 64 * NT;
  static constexpr int G_AT = BR * M::TRS, ST_AT = 2 * G_AT;    // both tiles are read in rows and transposed
  static constexpr int K_AT = ST_AT + 3 * BR * 4;               // GQ: the block's keys,
  static constexpr int DS_AT = K_AT + KEYS * M::TRS;            // each wavefront's score gradients of CH keys as (key, row),
  static constexpr int DS_ROW = M::CH * M::SZ + (M::WIDE ? 16 : 32), DS_WAVE = M::CH * DS_ROW;
  static constexpr int RED_AT = DS_AT + 4 * DS_WAVE;            // and its share of gq of the tile's rows, float32
  static constexpr int RED_ROW = DP + 4;
  static constexpr int LDS = GQ ? RED_AT + 4 * BR * RED_ROW * 4 : K_AT;
  static constexpr int NP = (BR * M::PPR + 255) / 256;
  // behind them, with a (query, key) mask: a bit per row and key, 16 keys of a row in a word, the words of a key tile's rows side by side.
  // A thread loads 16 keys of a row at a time, with the rows' next tile (7 x 197 x 1062 x 32 heads of 24, bf16: 88 us; every lane
  // its own bytes from the lines of four rows, two key tiles each: 111)
  static constexpr int CELLS = (BR * 4 * NT + 255) / 256, MASK = 2 * BR * 4 * NT, DROP = 4 * BR;   // DROP: the rows' dropout hashes
  // P of a normalised row is about 1 / S: in float16 it is scaled by 2^14 (the largest power of two whose product with 1 is finite
  // with room to spare) so that probabilities down to 2^-28 keep their 11 bits; exact to undo
  // Score gradients are rounded as they are: they follow grad_out's size, which a loss scale sets, down to float16's 2^-25 absolute
  static constexpr float P_SCALE = TY == DI_F16 ? 16384.f : 1.f, P_LOG2 = TY == DI_F16 ? 14.f : 0.f;
};

struct __attribute__((packed)) MaskCell {
  u4 v;
};

// FULL: with a (query, key) mask, dropout, or few keys (the test in the other variant's loop cost 1200 x 60 x 112 4 us of 78)
template <int TY, int DP, int NT, bool GQ, bool FULL>
__global__ __launch_bounds__(256, GQ && DP == 16 && !FULL ? 3 : DP >= 64 && TY != DI_F32 && FULL ? 2 : 1) void attention_gkv_kernel(Args a) {
  using C = GkvCfg<TY, DP, NT, GQ>;
  using M = Mm<TY, DP>;
  extern __shared__ __align__(16) char lds[];
  float *slse = reinterpret_cast<float *>(lds + C::ST_AT), *sdelta = slse + C::BR, *sone = sdelta + C::BR;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 15, g = lane >> 4;
  const Where at = where<true>(a);
  const int rows = a.G * a.L, nkeys = keys_of(a, at.b);
  const bool few = FULL && NT == (GQ ? 2 : 1) && a.S <= kFew;   // (few keys: the plan's smallest block)
  const int key0 = at.blk * C::KEYS;
  // a block without keys: zeros (the only block: gq's zeros, too)
  const int r0 = at.sp * a.range, r1 = key0 < nkeys || (GQ && a.blocks == 1) ? min(r0 + a.range, rows) : r0;
  const bool whole = key0 + C::KEYS <= nkeys && a.kmask == nullptr;
  const int waves = min(4, max(1, (nkeys - key0 + 16 * NT - 1) / (16 * NT)));             // wavefronts with keys
  const long long row_id = ((long long)at.b * a.Hk + at.hk) * rows;
  const char *kb = a.k + at.b * a.k_bs + (long long)at.hk * a.D * M::SZ, *vb = a.v + at.b * a.v_bs + (long long)at.hk * a.D * M::SZ;

  // rows of Q and go as KeyStage holds keys; a tile that lies in one head has a uniform base
  constexpr int STEP = 256 / M::PPR;
  u4 qs[C::NP], gs[C::NP], os[C::NP];                           // os: GQ forms delta from the forward's output
  float ls = INFINITY, de = 0.f;
  u4 cells[C::CELLS];                                           // the mask of one row and 16 keys each
  bool empty[C::NP];                                            // (query, key) mask: rows that it leaves without keys become zeros, so that
                                                                // what they hold - a NaN - meets no product over the rows
  const int piece = tid % M::PPR, first = tid / M::PPR;
  const bool in = piece * 16 < a.D * M::SZ && (C::BR >= STEP || first < C::BR);
  const unsigned qo = (unsigned)(first * a.q_rs) + piece * 16, go = (unsigned)(first * a.go_rs) + piece * 16;
  const char *qb = a.q + at.b * a.q_bs, *gb = a.go + at.b * a.go_bs;
  const long long o_rs = (long long)a.Hk * a.G * a.D * M::SZ;
  const unsigned oo = (unsigned)(first * o_rs) + piece * 16;
  const char *ob = a.o + (long long)at.b * a.L * o_rs;
  auto fetch = [&](int t0) {
    const int head0 = a.G == 1 ? 0 : (int)a.by_L.of(t0), l0 = t0 - head0 * a.L;
    if (t0 + C::BR <= r1 && l0 + C::BR <= a.L) {
      const long long col = (long long)(at.hk * a.G + head0) * a.D * M::SZ;
      const char *qt = qb + l0 * a.q_rs + col, *gt = gb + l0 * a.go_rs + col, *ot = ob + l0 * o_rs + col;
#pragma unroll
      for (int j = 0; j < C::NP; ++j) {
        qs[j] = gs[j] = os[j] = u4{0, 0, 0, 0};
        if (in) {
          qs[j] = *reinterpret_cast<const u4 *>(qt + j * STEP * a.q_rs + qo);
          gs[j] = *reinterpret_cast<const u4 *>(gt + j * STEP * a.go_rs + go);
          if (GQ) os[j] = *reinterpret_cast<const u4 *>(ot + j * STEP * o_rs + oo);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < C::NP; ++j) {
        const int r = t0 + first + j * STEP;
        qs[j] = gs[j] = os[j] = u4{0, 0, 0, 0};
        if (in && r < r1) {
          const int head = a.G == 1 ? 0 : (int)a.by_L.of(r), l = r - head * a.L;
          const long long col = (long long)(at.hk * a.G + head) * a.D * M::SZ + piece * 16;
          qs[j] = *reinterpret_cast<const u4 *>(qb + l * a.q_rs + col);
          gs[j] = *reinterpret_cast<const u4 *>(gb + l * a.go_rs + col);
          if (GQ) os[j] = *reinterpret_cast<const u4 *>(ob + l * o_rs + col);
        }
      }
    }
    if (FULL && a.allowed != nullptr) {
#pragma unroll
      for (int j = 0; j < C::CELLS; ++j) {
        const int e = tid + 256 * j, r = min(t0 + e / (4 * NT), rows - 1), head = a.G == 1 ? 0 : (int)a.by_L.of(r);
        const int at_key = key0 + 16 * (e % (4 * NT));
        const unsigned char *line = a.allowed + at.b * a.allowed_bs + (r - head * a.L) * a.allowed_rs;
        cells[j] = u4{0, 0, 0, 0};
        if (C::CELLS * 256 > C::BR * 4 * NT && e >= C::BR * 4 * NT) continue;
        if (a.S >= 16) {                                        // the row's last 16 keys: moved up when they become bits
          cells[j] = reinterpret_cast<const MaskCell *>(line + min(at_key, a.S - 16))->v;
        } else {                                                // (a single key block: the other key tiles' keys are not there)
#pragma unroll
          for (int k = 0; k < 4; ++k) cells[j][k] = look<true>(line, 4 * k, a.S);
        }
      }
#pragma unroll
      for (int j = 0; j < C::NP; ++j) {
        const int r = t0 + first + j * STEP;
        empty[j] = r < r1 && a.lse[row_id + r] == -INFINITY;
      }
    }
    if (tid < C::BR) {
      const bool ok = t0 + tid < r1;
      ls = ok ? a.lse[row_id + t0 + tid] : INFINITY;
      if (!GQ) de = ok ? a.delta[row_id + t0 + tid] : 0.f;
    }
  };
  if (r0 < r1) fetch(r0);

  typename M::RF kf[NT][M::NK], vf[NT][M::NK];
  f4 gk[NT][M::ND], gv[NT][M::ND];
  bool valid[NT];
  int key[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    key[n] = key0 + (wave * NT + n) * 16 + i;
    valid[n] = key[n] < nkeys && (a.kmask == nullptr || a.kmask[at.b * a.kmask_bs + key[n]] != 0);
#pragma unroll
    for (int kk = 0; kk < M::NK; ++kk) {
      kf[n][kk] = M::row_frag_of(kb + key[n] * a.k_rs, kk, g, a.D, valid[n]);
      vf[n][kk] = M::row_frag_of(vb + key[n] * a.v_rs, kk, g, a.D, valid[n]);
    }
#pragma unroll
    for (int d = 0; d < M::ND; ++d) gk[n][d] = gv[n][d] = f4{0.f, 0.f, 0.f, 0.f};
  }
  const unsigned long long seed = FULL && a.drop ? seed_of(a) : 0;
  if constexpr (GQ) {                                           // the keys once more, for the products that contract over them
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int kk = 0; kk < M::NK; ++kk) M::put_x(lds + C::K_AT + ((wave * NT + n) * 16 + i) * M::TRS, kk, g, i, kf[n][kk]);
  }

  for (int t0 = r0; t0 < r1; t0 += C::BR) {
    __syncthreads();
    if (C::BR >= STEP || first < C::BR) {
#pragma unroll
      for (int j = 0; j < C::NP; ++j) {
        if (FULL && a.allowed != nullptr && empty[j]) qs[j] = gs[j] = os[j] = u4{0, 0, 0, 0};
        const int at_row = (first + j * STEP) * M::TRS + ((piece * 16) ^ M::x(first + j * STEP));
        if (M::whole(piece)) {
          *reinterpret_cast<u4 *>(lds + at_row) = qs[j];
          *reinterpret_cast<u4 *>(lds + C::G_AT + at_row) = gs[j];
        }
        if (GQ) {
          float d = M::widen_dot({gs[j]}, {os[j]});
#pragma unroll
          for (int x = 1; x < M::PPR; x *= 2) d += __shfl_xor(d, x);
          if (piece == 0) sdelta[first + j * STEP] = d * (1.f / C::P_SCALE);
        }
      }
    }
    if (FULL && a.allowed != nullptr) {
#pragma unroll
      for (int j = 0; j < C::CELLS; ++j) {
        const int e = tid + 256 * j;
        unsigned bits = 0;
        if (a.S < 16) {
#pragma unroll
          for (int k = 0; k < 4; ++k) cells[j][k] = moved<true>(cells[j][k], 4 * k, a.S);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {                           // bytes != 0 -> their top bits -> four adjacent bits (no two of the product's terms meet)
          const unsigned w = cells[j][k], top = (((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w) & 0x80808080u;
          bits |= ((top >> 7) * 0x01020408u >> 24 & 0xfu) << (4 * k);
        }
        if (C::CELLS * 256 > C::BR * 4 * NT && e >= C::BR * 4 * NT) continue;
        const int at_key = key0 + 16 * (e % (4 * NT)), up = a.S >= 16 ? min(max(at_key - (a.S - 16), 0), 16) : 0;
        *reinterpret_cast<unsigned short *>(lds + C::LDS + 2 * ((e % (4 * NT)) * C::BR + e / (4 * NT))) = (unsigned short)(bits >> up);
      }
    }
    if (tid < C::BR) {
      slse[tid] = ls == -INFINITY ? INFINITY : ls - C::P_LOG2;
      if (!GQ) sdelta[tid] = de * (1.f / C::P_SCALE);
      if (few) {
        const int r = min(t0 + tid, rows - 1), head = a.G == 1 ? 0 : (int)a.by_L.of(r);
        sone[tid] = one_key(a, at.b, r - head * a.L, nkeys) ? 0.f : 1.f;
      }
      if (FULL && a.drop) *reinterpret_cast<unsigned *>(lds + C::LDS + C::MASK + 4 * tid) = drop_row(seed, row_id + t0 + tid);
    }
    __syncthreads();
    if (t0 + C::BR < r1) fetch(t0 + C::BR);
#pragma unroll 1
    for (int rc = 0; rc < C::BR; rc += M::CH) {
      if (t0 + rc >= r1 || (GQ && wave >= waves)) break;
      typename M::PF pf[NT], df[NT];
      typename M::TF gt_[M::ND];
#pragma unroll
      for (int u = 0; u < M::NT; ++u) {
        f4 s[NT], dp[NT];
        unsigned keep[NT];                                      // dropout: bit 4 r = row 4 g + r keeps the lane's key
        if (FULL && a.drop) {
          // four lanes share four keys: lane j of them hashes row 4 g + j's four numbers, the four rows' decisions are put together (2 x 200 x
          // 32 400 x 8 heads of 16, half precision: 166 us; every lane its four rows' numbers, 236; without dropout 66)
          const unsigned dr = *reinterpret_cast<const unsigned *>(lds + C::LDS + C::MASK + 4 * (rc + 16 * u + 4 * g + (i & 3)));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const unsigned k4 = (unsigned)key[n] >> 2, x = drop_pair(dr, k4, false), y = drop_pair(dr, k4, true);
            unsigned w = ((x & 0xffffu) >= a.drop ? 1u : 0u) | ((x >> 16) >= a.drop ? 2u : 0u) | ((y & 0xffffu) >= a.drop ? 4u : 0u) |
                         ((y >> 16) >= a.drop ? 8u : 0u);
            w <<= 4 * (i & 3);
            w |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)w, 0xb1, 0xf, 0xf, true);       // lanes 1 0 3 2
            w |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)w, 0x4e, 0xf, 0xf, true);       // lanes 2 3 0 1
            keep[n] = w >> (i & 3);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n] = dp[n] = f4{0.f, 0.f, 0.f, 0.f};
        typename M::RF qf[M::NK], gf[M::NK];                    // the tile's fragments before its first product
#pragma unroll
        for (int kk = 0; kk < M::NK; ++kk) {
          qf[kk] = M::row_frag_x(lds + (rc + 16 * u + i) * M::TRS, kk, g, i);
          gf[kk] = M::row_frag_x(lds + C::G_AT + (rc + 16 * u + i) * M::TRS, kk, g, i);
        }
        if (!GQ) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < M::NK; ++kk)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            s[n] = M::dot(qf[kk], kf[n][kk], s[n]);
            dp[n] = M::dot(gf[kk], vf[n][kk], dp[n]);
          }
        const f4 l4 = *reinterpret_cast<const f4 *>(slse + rc + 16 * u + 4 * g), d4 = *reinterpret_cast<const f4 *>(sdelta + rc + 16 * u + 4 * g);
        if (!GQ && u == M::NT - 1) {                            // go^T in flight behind the last exponentials
#pragma unroll
          for (int d = 0; d < M::ND; ++d) gt_[d] = M::tr_frag(lds + C::G_AT, M::TRS, rc, d, i, g);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (FULL && a.allowed != nullptr) {                   // bit i of the words of rows 4 g .. + 3
            const u2 may = *reinterpret_cast<const u2 *>(lds + C::LDS + 2 * ((wave * NT + n) * C::BR + rc + 16 * u + 4 * g));
#pragma unroll
            for (int r = 0; r < 4; ++r) s[n][r] = (may[r >> 1] >> (16 * (r & 1) + i) & 1u) != 0 ? s[n][r] : -INFINITY;
          }
          f4 p, ds;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // (a column is one key: whatever the column of an excluded key holds stays there, and is dropped at the end)
            // pr = P_SCALE p, ds = pr ((dp - delta) / P_SCALE): the scale sits in the rows' two numbers
            const float pr = __builtin_amdgcn_exp2f(fmaf(s[n][r], a.scale2, -l4[r]));
            if (FULL && a.drop) {
              const bool kept = (keep[n] >> (4 * r) & 1u) != 0;
              p[r] = kept ? pr : 0.f;                        // the kept ones' scale: at the end
              dp[n][r] = kept ? dp[n][r] * a.keep_scale : 0.f;
            } else {
              p[r] = pr;
            }
            ds[r] = pr * fmaf(dp[n][r], 1.f / C::P_SCALE, -d4[r]);
          }
          if (few) ds *= *reinterpret_cast<const f4 *>(sone + rc + 16 * u + 4 * g);
          if (GQ && !whole) {                                   // gq sums over the columns: those of excluded keys have to be zero
#pragma unroll
            for (int r = 0; r < 4; ++r) ds[r] = valid[n] ? ds[r] : 0.f;
          }
          M::pack(pf[n], u, p);
          M::pack(df[n], u, ds);
        }
      }
      auto by_rows = [&]() {                                    // gv^T += go^T P, gk^T += Q^T dS
#pragma unroll
        for (int d = 0; d < M::ND; ++d) {
          const typename M::TF gt = GQ ? M::tr_frag(lds + C::G_AT, M::TRS, rc, d, i, g) : gt_[d];
#pragma unroll
          for (int n = 0; n < NT; ++n) gv[n][d] = M::acc(gt, pf[n], gv[n][d]);
        }
#pragma unroll
        for (int d = 0; d < M::ND; ++d) {
          const typename M::TF qt = M::tr_frag(lds, M::TRS, rc, d, i, g);
#pragma unroll
          for (int n = 0; n < NT; ++n) gk[n][d] = M::acc(qt, df[n], gk[n][d]);
        }
      };
      if constexpr (!GQ) by_rows();
      if constexpr (GQ) {
        // gq^T = K^T dS^T of the wavefront's keys, CH of them at a time: dS leaves as (key, row) rows of the wavefront's own buffer - a lane
        // holds four rows of one key - and comes back transposed as the operand; LDS serves a wavefront in order, no barrier
        char *mine = lds + C::DS_AT + wave * C::DS_WAVE;
        f4 gq[M::NT][M::ND];
#pragma unroll
        for (int u = 0; u < M::NT; ++u)
#pragma unroll
          for (int d = 0; d < M::ND; ++d) gq[u][d] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NT / M::NT; ++c) {
#pragma unroll
          for (int h = 0; h < M::NT; ++h) {
            const int n = c * M::NT + h;
            char *at_key = mine + (16 * h + i) * C::DS_ROW + ((4 * g * M::SZ) ^ M::x(i));
            if constexpr (M::WIDE) {
              *reinterpret_cast<u4 *>(at_key) = df[n].v;
            } else {
              *reinterpret_cast<u2 *>(at_key) = u2{df[n].v[0], df[n].v[1]};
              *reinterpret_cast<u2 *>(at_key + 32) = u2{df[n].v[2], df[n].v[3]};
            }
          }
          __builtin_amdgcn_wave_barrier();
          if (c == 0) by_rows();                                // products in the shadow of the first round trip
#pragma unroll
          for (int u = 0; u < M::NT; ++u) {
            const typename M::PF st = {M::tr_frag(mine, C::DS_ROW, 0, u, i, g).v};
#pragma unroll
            for (int d = 0; d < M::ND; ++d)
              gq[u][d] = M::acc(M::tr_frag(lds + C::K_AT, M::TRS, wave * 16 * NT + c * M::CH, d, i, g), st, gq[u][d]);
          }
          __builtin_amdgcn_wave_barrier();
        }
        float *red = reinterpret_cast<float *>(lds + C::RED_AT) + (wave * C::BR + rc) * C::RED_ROW;
#pragma unroll
        for (int u = 0; u < M::NT; ++u)
#pragma unroll
          for (int d = 0; d < M::ND; ++d) *reinterpret_cast<f4 *>(red + (16 * u + i) * C::RED_ROW + 16 * d + 4 * g) = gq[u][d];
      }
    }
    if constexpr (GQ) {                                         // the wavefronts' shares of the tile's gq
      __syncthreads();
      const float *red = reinterpret_cast<const float *>(lds + C::RED_AT);
      for (int e = tid; e < C::BR * (DP / 4); e += 256) {
        const int rr = e / (DP / 4), d = 4 * (e % (DP / 4)), r = t0 + rr;
        if (r >= r1 || d >= a.D) continue;
        f4 x = *reinterpret_cast<const f4 *>(red + rr * C::RED_ROW + d);
        for (int w = 1; w < waves; ++w) x += *reinterpret_cast<const f4 *>(red + (w * C::BR + rr) * C::RED_ROW + d);
        if (a.blocks > 1) {
          *reinterpret_cast<f4 *>(a.part + ((long long)at.blk * a.B * a.Hk * rows + row_id + r) * a.D + d) = x;
        } else {
          const int head = a.G == 1 ? 0 : (int)a.by_L.of(r);
          M::store4(a.gq + (((long long)at.b * a.L + (r - head * a.L)) * o_rs) + ((at.hk * a.G + head) * a.D + d) * M::SZ, x * a.scale);
        }
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if (key[n] >= a.S) continue;
    if (!valid[n]) {
#pragma unroll
      for (int d = 0; d < M::ND; ++d) gk[n][d] = gv[n][d] = f4{0.f, 0.f, 0.f, 0.f};
    }
    if (a.splits > 1) {
      const long long rec = (((long long)at.sp * a.B + at.b) * a.Hk + at.hk) * a.S + key[n];
#pragma unroll
      for (int d = 0; d < M::ND; ++d)
        if (16 * d + 4 * g < a.D) {
          *reinterpret_cast<f4 *>(a.part_k + rec * a.D + 16 * d + 4 * g) = gk[n][d];
          *reinterpret_cast<f4 *>(a.part_v + rec * a.D + 16 * d + 4 * g) = gv[n][d];
        }
    } else {
      const long long col = (long long)at.hk * a.D * M::SZ;
      char *pk = a.gk + at.b * a.gk_bs + key[n] * a.gk_rs + col, *pv = a.gv + at.b * a.gv_bs + key[n] * a.gv_rs + col;
#pragma unroll
      for (int d = 0; d < M::ND; ++d)
        if (16 * d + 4 * g < a.D) {
          M::store4(pk + (16 * d + 4 * g) * M::SZ, gk[n][d] * a.scale);
          M::store4(pv + (16 * d + 4 * g) * M::SZ, gv[n][d] * (a.keep_scale / C::P_SCALE));
        }
    }
  }
}

template <int TY>
__global__ __launch_bounds__(256) void attention_gkv_join_kernel(Args a) {
  using M = Mm<TY, 16>;
  const int q4 = a.D / 4;
  const long long all = (long long)a.B * a.Hk * a.S, id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= all * q4) return;
  const long long rid = id / q4;
  const int d = 4 * (int)(id % q4), s = (int)(rid % a.S), hk = (int)(rid / a.S % a.Hk), b = (int)(rid / a.S / a.Hk);
  f4 k = {0.f, 0.f, 0.f, 0.f}, v = k;
  for (int r = 0; r < a.splits; ++r) {
    k += *reinterpret_cast<const f4 *>(a.part_k + (r * all + rid) * a.D + d);
    v += *reinterpret_cast<const f4 *>(a.part_v + (r * all + rid) * a.D + d);
  }
  const long long col = ((long long)hk * a.D + d) * M::SZ;
  M::store4(a.gk + b * a.gk_bs + s * a.gk_rs + col, k * a.scale);
  M::store4(a.gv + b * a.gv_bs + s * a.gv_rs + col, v * (a.keep_scale / GkvCfg<TY, 16, 2, true>::P_SCALE));
}

}  // namespace at
}  // namespace di
