// Forward of the attention to another sequence.  Per row:  s_j = scale q . k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),
// one pass over the keys with the running maximum m and sum.
//
// S^T = K Q^T (16 keys x 16 rows a tile: a row is a lane's column, its running maximum and sum are two registers), O^T += V^T P^T
// with the exponentials' registers as the operand.  The keys' tile goes through LDS (loads of the next one in flight in registers
// behind the products), where four wavefronts read it: WQ = 4 wavefronts with MT row tiles each on the same keys, or - up to 16
// rows, single queries - WQ = 1, four wavefronts on four parts of the tile, joined at the end.  Few row blocks: the keys are split
// over workgroups, which leave (m, sum, O) in float32 for a second launch to join.
//
// The maximum is corrected only when a score exceeds it by more than 8 (a factor of 256 in exp2's argument, harmless in float32 and
// in the 16-bit probabilities): the test is one comparison per tile against the lane's own scores, the exchange between lanes and
// the correction of the sums run when any lane asks for them - a few times per row, not once per tile.  `m` is what the exponents are
// taken from: the maximum, for float16 less 7 - with the 8 above, probabilities of up to 2^15 (65 504 is the type's largest), their rounding
// stays relative down to 2^-21 of the largest and reaches zero at 2^-32, where the float32 sum beside them would still count them at 2^-25.
//
// What bounds it, and what it measured (shares of the SIMDs' cycles from the counters of the final build):
//   heads of 128 and 64 (2048 x 8192 x 16 heads of 128, bf16: 180 us = 765 TFLOP/s, a large matrix product reaches 1085 on this card): the
//     matrix cores work in 40 % of the cycles, the vector unit in 44, LDS in 40; two wavefronts a SIMD, each of which alternates products and
//     exponentials, overlap them in part and wait 43 % of their time for a unit to take their next instruction
//   heads of 16: a pair of row and key costs 32 multiply-adds, an exponential and five vector instructions.  Float32 (200 x 32 400 x 8, 49 us
//     = 68 TFLOP/s of 149): matrix cores 53 %, vector unit 29, overlapped in part.  Half precision, 2 samples (37 us): vector unit 61 %,
//     matrix cores 13.  Writing float32 operands as three bf16 parts would take the products of a tile from 256 to 96 cycles and the
//     vector instructions from 160 to 256 (six more a probability): 416 -> 352 where nothing overlaps, a loss where everything does; not built
//   single queries (16 samples of up to 32 768 keys x 8 key heads of 128, 1.07 GB): the memory, 190 us = 5.6 TB/s
// Spilled registers: with masks and dropout the 16-bit kernels of 32 dims keep 2 - 6 and those of 128 dims 8 of their lanes' values in scratch
// (12 - 36 bytes, at the bound of two wavefronts a SIMD); every other variant none.  1024 x 4096, 8 heads, bf16, with a (query, key) mask against
// without: 32 dims 36.1 and 27.5 us, 64 (no spills) 37.9 and 30.2, 128 47.6 and 38.0 - the mask's own instructions in all three.
#pragma once
#include <type_traits>

#include "attention.h"

namespace di {
namespace at {

template <int TY, int DP, int MT, int WQ>
struct FwdCfg {
  using M = Mm<TY, DP>;
  static constexpr int WK = 4 / WQ;
  static constexpr int CPT = WQ == 1 ? 1 : 64 / M::CH;          // chunks of CH keys per wavefront and tile
  static constexpr int TILE = WK * CPT * M::CH;
  static constexpr int V_AT = TILE * M::ROWS, BIAS_AT = V_AT + TILE * M::TRS;
  static constexpr int JOIN = WQ == 1 ? 4 * 16 * (DP + 2) * 4 : 0;
  static constexpr int LDS = BIAS_AT + TILE * 4 > JOIN ? BIAS_AT + TILE * 4 : JOIN;
  static constexpr int ROWS_PER_BLOCK = 16 * MT * WQ;
  static constexpr int NP = (TILE * M::PPR + 255) / 256;        // pieces per thread, K and V each
  static constexpr float P_LOG2 = TY == DI_F16 ? 7.f : 0.f;     // the scale of the probabilities in `o` and `l` alike
};

// The staged loads of a tile of keys: rows t0 .. of K and V, zeros where there is no key (so that no NaN of an excluded key or of
// memory behind the last one reaches a product).  Thread e holds piece e % PPR of the rows e / PPR + j 256 / PPR: a uniform base per
// tile and j, and one 32-bit lane offset each for K and V that never changes.
template <class C>
struct KeyStage {
  using M = typename C::M;
  static constexpr int STEP = 256 / M::PPR;                     // rows per piece index j
  u4 k[C::NP], v[C::NP];
  unsigned char part[C::NP];                                    // with a key mask: whether the key takes part
  unsigned ko, vo;
  int key;
  bool in;                                                      // the piece lies within the head dim (and the tile)
  __device__ __forceinline__ void init(const Args &a) {
    const int p = threadIdx.x % M::PPR;
    key = threadIdx.x / M::PPR;
    ko = (unsigned)(key * a.k_rs) + p * 16;
    vo = (unsigned)(key * a.v_rs) + p * 16;
    in = p * 16 < a.D * M::SZ && (C::TILE >= STEP || key < C::TILE);
  }
  __device__ __forceinline__ void fetch(const Args &a, const char *kb, const char *vb, const unsigned char *km, int t0, int k1) {
    const char *kt = kb + t0 * a.k_rs, *vt = vb + t0 * a.v_rs;
    if (km == nullptr && t0 + C::TILE <= k1) {
#pragma unroll
      for (int j = 0; j < C::NP; ++j) {
        k[j] = v[j] = u4{0, 0, 0, 0};
        if (in) {
          k[j] = *reinterpret_cast<const u4 *>(kt + j * STEP * a.k_rs + ko);
          v[j] = *reinterpret_cast<const u4 *>(vt + j * STEP * a.v_rs + vo);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < C::NP; ++j) {
        const int s = t0 + key + j * STEP;
        k[j] = v[j] = u4{0, 0, 0, 0};
        if (km != nullptr) part[j] = km[min(s, k1 - 1)];
        if (in && s < k1) {                                     // (masked keys are loaded, too: the loads do not wait for the mask)
          k[j] = *reinterpret_cast<const u4 *>(kt + j * STEP * a.k_rs + ko);
          v[j] = *reinterpret_cast<const u4 *>(vt + j * STEP * a.v_rs + vo);
        }
      }
    }
  }
  // KX / VX: the tile of K / V is a TRS tile
  template <bool KX, bool VX>
  __device__ __forceinline__ void commit(char *lds, int v_at, bool masked) {
    const int p = threadIdx.x % M::PPR;
    if (C::TILE >= STEP || key < C::TILE) {
#pragma unroll
      for (int j = 0; j < C::NP; ++j) {
        const int row = key + j * STEP, x = M::x(row);
        if (masked && part[j] == 0) k[j] = v[j] = u4{0, 0, 0, 0};
        if (!M::whole(p)) continue;
        *reinterpret_cast<u4 *>(lds + row * (KX ? M::TRS : M::ROWS) + ((p * 16) ^ (KX ? x : 0))) = k[j];
        *reinterpret_cast<u4 *>(lds + v_at + row * (VX ? M::TRS : M::ROWS) + ((p * 16) ^ (VX ? x : 0))) = v[j];
      }
    }
  }
};

// max without the quieting of its operands (v_max_f32 x, x) that fmaxf needs for values that may be signalling NaN: two instructions less
// a score.  A NaN score loses the comparison but stays a NaN in the exponential.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, INFINITY); }

// 4 keys x 1 row of the (row, key) mask as the bytes of a word, one load wherever the row starts (53 x 721 x 651, 4 heads of 32, forward:
// four byte loads 430 us, one of a word 96).  EDGE: keys may lie behind the row's end - its last word is taken, which `exclude` moves up
// once it has arrived; what it then holds for those keys does not matter, they are excluded anyway.  A row that is not there reads the
// last one's mask.
struct __attribute__((packed)) MaskWord {
  unsigned w;
};
template <bool EDGE>
__device__ __forceinline__ unsigned look(const unsigned char *row, int key, int S) {
  if (!EDGE) return reinterpret_cast<const MaskWord *>(row + key)->w;
  if (S >= 4) return reinterpret_cast<const MaskWord *>(row + min(key, S - 4))->w;
  unsigned w = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r) w |= (unsigned)row[min(key + r, S - 1)] << (8 * r);
  return w;
}
template <bool EDGE>
__device__ __forceinline__ unsigned moved(unsigned w, int key, int S) {
  return EDGE && S >= 4 ? w >> (8 * min(max(key - (S - 4), 0), 3)) : w;
}
__device__ __forceinline__ void exclude(unsigned w, f4 &s) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if ((w >> (8 * r) & 0xffu) == 0) s[r] = -INFINITY;
}

// FULL: with a key mask, a (query, key) mask or dropout; without them only the last tile of a range is tested key by key
template <int TY, int DP, int MT, int WQ, bool FULL>
__global__ __launch_bounds__(256, (DP >= 96 && TY != DI_F32) || (DP == 32 && FULL) ? 2 : 1) void attention_fwd_kernel(Args a) {
  using C = FwdCfg<TY, DP, MT, WQ>;
  using M = Mm<TY, DP>;
  extern __shared__ __align__(16) char lds[];
  float *bias = reinterpret_cast<float *>(lds + C::BIAS_AT);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
  const Where at = where<false>(a);
  // the wavefront that gets one row tile more than the others is not the same SIMD's in every workgroup
  const int wq = WQ == 1 ? 0 : (wave + at.sp + at.hk + at.b) % WQ, wk = wave / WQ;
  const int rows = a.G * a.L, ntile = (rows + 15) / 16;
  const int k0 = at.sp * a.range, k1 = min(k0 + a.range, keys_of(a, at.b));
  if (a.splits > 1 && k0 >= k1) return;                         // the join knows the sample's keys, too
  const char *kb = a.k + at.b * a.k_bs + (long long)at.hk * a.D * M::SZ, *vb = a.v + at.b * a.v_bs + (long long)at.hk * a.D * M::SZ;
  const unsigned char *km = !FULL || a.kmask == nullptr ? nullptr : a.kmask + at.b * a.kmask_bs;
  const long long row_id = ((long long)at.b * a.Hk + at.hk) * rows;

  typename M::RF qf[MT][M::NK];
  f4 o[MT][M::ND];
  float m[MT], l[MT];
  int row[MT], query[MT];
  unsigned drow[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int tile = (at.blk * MT + t) * WQ + wq;               // row tiles dealt out to the wavefronts in turn
    row[t] = tile < ntile ? 16 * tile + i : rows;
    const int r = min(row[t], rows - 1), head = a.G == 1 ? 0 : (int)a.by_L.of(r);
    query[t] = r - head * a.L;
    const char *qp = a.q + at.b * a.q_bs + query[t] * a.q_rs + (long long)(at.hk * a.G + head) * a.D * M::SZ;
#pragma unroll
    for (int kk = 0; kk < M::NK; ++kk) qf[t][kk] = M::row_frag_of(qp, kk, g, a.D, row[t] < rows);
#pragma unroll
    for (int d = 0; d < M::ND; ++d) o[t][d] = f4{0.f, 0.f, 0.f, 0.f};
    m[t] = kLowest;
    l[t] = 0.f;
    drow[t] = FULL && a.drop ? drop_row(seed_of(a), row_id + r) : 0;
  }

  // one tile of keys for the wavefront's first N row tiles; EDGE: keys are tested
  auto tile = [&](auto edge, auto count, int t0) {
    constexpr bool EDGE = decltype(edge)::value;
    constexpr int N = decltype(count)::value;
#pragma unroll
    for (int c = 0; c < C::CPT; ++c) {
      const int kc = (wk * C::CPT + c) * M::CH;                 // first key of the chunk in the tile
      if (EDGE && t0 + kc >= k1) break;
      unsigned may[MT][M::NT];                                  // in flight behind the products
      if (FULL && a.allowed != nullptr) {
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
          for (int u = 0; u < M::NT; ++u)
            may[t][u] = look<EDGE>(a.allowed + at.b * a.allowed_bs + query[t] * a.allowed_rs, t0 + kc + 16 * u + 4 * g, a.S);
      }
      typename M::RF kf[M::NT][M::NK];                          // all of the chunk's before its first product: one wait, not one each
#pragma unroll
      for (int u = 0; u < M::NT; ++u)
#pragma unroll
        for (int kk = 0; kk < M::NK; ++kk) kf[u][kk] = M::row_frag(lds + (kc + 16 * u + i) * M::ROWS, kk, g);
      __builtin_amdgcn_sched_barrier(0);
      f4 s[MT][M::NT];
#pragma unroll
      for (int u = 0; u < M::NT; ++u) {
#pragma unroll
        for (int t = 0; t < N; ++t) s[t][u] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < M::NK; ++kk)
#pragma unroll
          for (int t = 0; t < N; ++t) s[t][u] = M::dot(kf[u][kk], qf[t][kk], s[t][u]);
        if (EDGE) {
          const f4 bb = *reinterpret_cast<const f4 *>(bias + kc + 16 * u + 4 * g);
#pragma unroll
          for (int t = 0; t < N; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[t][u][r] = bb[r] == 0.f ? s[t][u][r] : -INFINITY;
        }
        if (FULL && a.allowed != nullptr) {
#pragma unroll
          for (int t = 0; t < N; ++t) exclude(moved<EDGE>(may[t][u], t0 + kc + 16 * u + 4 * g, a.S), s[t][u]);
        }
      }
      float mx[MT];
      bool over = false;
#pragma unroll
      for (int t = 0; t < N; ++t) {
        mx[t] = kLowest;
#pragma unroll
        for (int u = 0; u < M::NT; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx[t] = larger(s[t][u][r], mx[t]);
        mx[t] *= a.scale2;
        over |= mx[t] > m[t] + (8.f + C::P_LOG2);
      }
      if (__any(over)) {
#pragma unroll
        for (int t = 0; t < N; ++t) {
          float x = fmaxf(mx[t], __shfl_xor(mx[t], 16));
          x = fmaxf(x, __shfl_xor(x, 32));
          x = fmaxf(x - C::P_LOG2, m[t]);
          const float f = __builtin_amdgcn_exp2f(m[t] - x);
          m[t] = x;
          l[t] *= f;
#pragma unroll
          for (int d = 0; d < M::ND; ++d) o[t][d] *= f;
        }
      }
      typename M::TF vf[M::ND];                                 // in flight behind the exponentials
#pragma unroll
      for (int d = 0; d < M::ND; ++d) vf[d] = M::tr_frag(lds + C::V_AT, M::TRS, kc, d, i, g);
      __builtin_amdgcn_sched_barrier(0);
      typename M::PF pf[MT];
#pragma unroll
      for (int t = 0; t < N; ++t) {
        f4 p[M::NT];
#pragma unroll
        for (int u = 0; u < M::NT; ++u) {
#pragma unroll
          for (int r = 0; r < 4; ++r) p[u][r] = __builtin_amdgcn_exp2f(fmaf(s[t][u][r], a.scale2, -m[t]));
          l[t] += (p[u][0] + p[u][1]) + (p[u][2] + p[u][3]);
          if (FULL && a.drop) {
            const unsigned k4 = (unsigned)(t0 + kc + 16 * u + 4 * g) >> 2;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const unsigned x = drop_pair(drow[t], k4, h);
              p[u][2 * h] = (x & 0xffffu) >= a.drop ? p[u][2 * h] : 0.f;      // the kept ones' scale: at the end
              p[u][2 * h + 1] = (x >> 16) >= a.drop ? p[u][2 * h + 1] : 0.f;
            }
          }
          M::pack(pf[t], u, p[u]);
        }
      }
#pragma unroll
      for (int d = 0; d < M::ND; ++d)
#pragma unroll
        for (int t = 0; t < N; ++t) o[t][d] = M::acc(vf[d], pf[t], o[t][d]);
    }
  };

  // row tiles that are there: absent ones are left out where a wavefront has four (200 rows x 32 400 of 16 dims: float32 52 -> 49 us, half
  // 37.9 -> 37.0); with two, the second copy of the loop cost more than it saved (511 x 4100 of 64 dims: 45 -> 50)
  const int first = at.blk * MT * WQ + wq, mine = first < ntile ? min(MT, (ntile - first + WQ - 1) / WQ) : 0;

  KeyStage<C> st;
  st.init(a);
  if (k0 < k1) st.fetch(a, kb, vb, km, k0, k1);
  auto step = [&](auto edge, int t0) {
    __syncthreads();                                            // the last tile's reads are done
    st.template commit<false, true>(lds, C::V_AT, km != nullptr);
    if (decltype(edge)::value && threadIdx.x < C::TILE) {
      const int s = t0 + threadIdx.x;
      bias[threadIdx.x] = s < k1 && (km == nullptr || km[s] != 0) ? 0.f : -INFINITY;
    }
    __syncthreads();
    if (t0 + C::TILE < k1) st.fetch(a, kb, vb, km, t0 + C::TILE, k1);
    if (MT <= 2 || mine == MT) tile(edge, std::integral_constant<int, MT>(), t0);
    else if (mine == MT - 1) tile(edge, std::integral_constant<int, (MT > 2 ? MT - 1 : 1)>(), t0);
    else if (mine > 0) tile(edge, std::integral_constant<int, (MT > 2 ? MT - 2 : 1)>(), t0);
  };
  int t0 = k0;
  if (km == nullptr)
    for (; t0 + C::TILE <= k1; t0 += C::TILE) step(std::false_type(), t0);
  for (; t0 < k1; t0 += C::TILE) step(std::true_type(), t0);
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    l[t] += __shfl_xor(l[t], 16);
    l[t] += __shfl_xor(l[t], 32);
  }

  if constexpr (WQ == 1) {                                      // join the four wavefronts (MT = 1)
    float *j = reinterpret_cast<float *>(lds);                  // (4, 16, DP + 2)
    __syncthreads();
    float *mine = j + (wave * 16 + i) * (DP + 2);
    if (g == 0) {
      mine[0] = m[0];
      mine[1] = l[0];
    }
#pragma unroll
    for (int d = 0; d < M::ND; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) mine[2 + 16 * d + 4 * g + r] = o[0][d][r];
    __syncthreads();
    if (wave != 0) return;
    float top = m[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, j[(w * 16 + i) * (DP + 2)]);
    l[0] = 0.f;
#pragma unroll
    for (int d = 0; d < M::ND; ++d) o[0][d] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float *p = j + (w * 16 + i) * (DP + 2);
      const float f = __builtin_amdgcn_exp2f(p[0] - top);
      l[0] = fmaf(p[1], f, l[0]);
#pragma unroll
      for (int d = 0; d < M::ND; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[0][d][r] = fmaf(p[2 + 16 * d + 4 * g + r], f, o[0][d][r]);
    }
    m[0] = top;
  }

#pragma unroll
  for (int t = 0; t < MT; ++t) {
    if (row[t] >= rows) continue;
    if (a.splits > 1) {
      const long long rec = (long long)at.sp * a.B * a.Hk * rows + row_id + row[t];
      if (g == 0) {
        a.part_ml[2 * rec] = m[t];
        a.part_ml[2 * rec + 1] = l[t];
      }
      float *p = a.part + rec * a.D;
#pragma unroll
      for (int d = 0; d < M::ND; ++d)
        if (16 * d + 4 * g < a.D) *reinterpret_cast<f4 *>(p + 16 * d + 4 * g) = o[t][d];
    } else {
      const float inv = l[t] == 0.f ? 0.f : a.keep_scale / l[t];         // an empty row: zeros
      if (a.lse != nullptr && g == 0) a.lse[row_id + row[t]] = l[t] == 0.f ? -INFINITY : m[t] + __builtin_amdgcn_logf(l[t]);
      const int head = a.G == 1 ? 0 : (int)a.by_L.of(row[t]);
      char *p = a.o + (((long long)at.b * a.L + query[t]) * a.Hk * a.G + at.hk * a.G + head) * a.D * M::SZ;
#pragma unroll
      for (int d = 0; d < M::ND; ++d)
        if (16 * d + 4 * g < a.D) M::store4(p + (16 * d + 4 * g) * M::SZ, o[t][d] * inv);
    }
  }
}

// The ranges' sums of a row joined: `group` lanes per row, 4 head dims a lane, the other lanes on further ranges, four ranges of a lane
// in flight (with their statistics).  by_unit: workgroups per (sample, key head).  STATS: forward, every range has its own maximum and
// sum; otherwise gq, plain sums.
template <int TY, bool STATS>
__global__ __launch_bounds__(256) void attention_join_kernel(Args a, int nd, int group) {
  using M = Mm<TY, 16>;
  const int lane = threadIdx.x % group, rows = a.G * a.L;
  const int pr = a.by_unit.of(blockIdx.x), b = a.by_hk.of(pr), hk = pr - b * a.Hk;
  const int r = (int)((blockIdx.x - pr * a.by_unit.d) * (256 / group) + threadIdx.x / group);
  if (r >= rows) return;                                        // whole groups leave: the exchanges below stay inside a group
  const long long all = (long long)a.B * a.Hk * rows, id = (long long)pr * rows + r;
  const int n = min(a.splits, (keys_of(a, b) + a.range - 1) / a.range);
  const int d = 4 * (lane % nd), step = group / nd;
  float top = kLowest, l = 0.f;
  f4 o = {0.f, 0.f, 0.f, 0.f};
  auto merge = [&](float m2, float l2, const f4 &o2) {
    const float x = fmaxf(top, m2), f = __builtin_amdgcn_exp2f(top - x), f2 = __builtin_amdgcn_exp2f(m2 - x);
    l = l * f + l2 * f2;
    o = o * f + o2 * f2;
    top = x;
  };
  for (int s0 = lane / nd; s0 < n; s0 += 4 * step) {
    f4 p[4];
    float m2[4], l2[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = s0 + u * step;
      p[u] = f4{0.f, 0.f, 0.f, 0.f};
      m2[u] = kLowest;
      l2[u] = 0.f;
      if (s < n) {
        if (d < a.D) p[u] = *reinterpret_cast<const f4 *>(a.part + (s * all + id) * a.D + d);
        if (STATS) {
          m2[u] = a.part_ml[2 * (s * all + id)];
          l2[u] = a.part_ml[2 * (s * all + id) + 1];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (STATS) merge(m2[u], l2[u], p[u]);
      else o += p[u];
    }
  }
  for (int x = nd; x < group; x *= 2) {
    f4 p;
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] = __shfl_xor(o[e], x);
    if (STATS) merge(__shfl_xor(top, x), __shfl_xor(l, x), p);
    else o += p;
  }
  if (STATS && a.lse != nullptr && lane == 0) a.lse[id] = l == 0.f ? -INFINITY : top + __builtin_amdgcn_logf(l);
  if (lane >= nd || d >= a.D) return;
  const int head = a.by_L.of(r);
  char *out = (STATS ? a.o : a.gq) + ((((long long)b * a.L + (r - head * a.L)) * a.Hk * a.G + hk * a.G + head) * a.D + d) * M::SZ;
  M::store4(out, o * (STATS ? (l == 0.f ? 0.f : a.keep_scale / l) : a.scale));
}

}  // namespace at
}  // namespace di
