// Attention of a set of queries to the states of another sequence: operand fragments, tiles and argument blocks shared by the
// forward (attention_fwd.h) and backward (attention_bwd.h) kernels.
//
// Rows.  The G query heads that share a key head are rows of one problem: row r < G L of (sample b, key head) is query r % L of
// head G hk + r / L.  lse / delta of (b, head, query) are then simply row r of a (B Hk, G L) matrix.
//
// Matrix instructions.  Every product is built from 16 x 16 tiles whose result has lane (i = lane % 16, g = lane / 16) hold
// column i, rows 4 g .. 4 g + 3.  Two forms of operand fragments:
//   row fragment: lane (i, g) holds row i's elements of the contraction over the head dim - 8 (32-wide products), 4 (16-wide,
//     head dim 16) 16-bit elements, or a float4 that feeds four 4-wide float32 products; the order inside a contraction is free,
//     so both operands simply use the same one and every fragment is one wide load;
//   transposed fragment: column 16 dt + i of the rows 4 g + r - the contraction runs over the tile's ROWS (keys or queries).
//     16-bit: two ds_read_b64_tr_b16 (two tiles of 16 rows, one 32-wide product); float32: four ds_read_b32.
// A result tile's registers are, as they are, the other operand of a product that contracts over its rows: the probabilities and
// score gradients never leave registers.
#pragma once
#include "di_common.h"

namespace di {
namespace at {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef short tr4 __attribute__((__vector_size__(4 * sizeof(short))));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.4028234663852886e38f;

__device__ __forceinline__ short to_half_bits(float x) { return __builtin_bit_cast(short, (_Float16)x); }
__device__ __forceinline__ short to_bf_bits(float x) { return __builtin_bit_cast(short, (__bf16)x); }

// TY: DI_F32 / DI_F16 / DI_BF16; DP: the head dim padded to 16, 32, 64, 96 or 128
template <int TY, int DP>
struct Mm {
  static constexpr bool WIDE = TY == DI_F32;
  static constexpr int SZ = WIDE ? 4 : 2;
  static constexpr int KD = WIDE || DP == 16 ? 16 : 32;         // head dims per row fragment
  static constexpr int NK = DP / KD, ND = DP / 16;
  static constexpr int CH = WIDE ? 16 : 32, NT = CH / 16;       // rows (keys / queries) per contraction over rows
  static constexpr int PPR = (DP == 96 ? 128 : DP) * SZ / 16;   // threads that stage a tile row's 16-byte pieces (a power of two)
  // tile row strides in bytes.  ROWS (read in rows only): + 16 keeps the fragments of 16 rows in different banks.  TRS (read transposed,
  // or both ways): float32 the same; 16-bit + 32, the stride that spreads the transposing reads of 8 rows over all banks.  Head dim 16 (no
  // padding): the two 16-byte pieces of every other 8 rows are exchanged (`x` on their offsets), which does the same for the 8-byte row
  // fragments (1200 x 60 x 112: conflicts 9.4 -> 3.9 million cycles); wider rows had no conflicts, and lost time to the addresses
  static constexpr int ROWS = DP * SZ + 16;
  static constexpr int TRS = WIDE ? DP * 4 + 16 : (DP == 16 ? 32 : DP * 2 + 32);
  struct RF {
    u4 v;
  };
  struct TF {
    u4 v;
  };
  struct PF {
    u4 v;
  };

  static __device__ __forceinline__ int x(int row) { return WIDE || DP != 16 ? 0 : (row & 8) << 1; }

  static __device__ __forceinline__ bool whole(int piece) { return DP != 96 || piece * 16 < DP * SZ; }   // the tile row has the piece
  static __device__ __forceinline__ int d0(int kk, int g) { return KD * kk + (WIDE || DP == 16 ? 4 : 8) * g; }
  static __device__ __forceinline__ RF row_frag(const char *row, int kk, int g) {
    RF f;
    if constexpr (!WIDE && DP == 16) {
      const u2 t = *reinterpret_cast<const u2 *>(row + 2 * d0(kk, g));
      f.v = u4{t[0], t[1], 0, 0};
    } else {
      f.v = *reinterpret_cast<const u4 *>(row + SZ * d0(kk, g));
    }
    return f;
  }
  // row i (mod 16) of a TRS tile
  static __device__ __forceinline__ RF row_frag_x(const char *row, int kk, int g, int i) {
    RF f;
    const char *at = row + ((SZ * d0(kk, g)) ^ x(i));
    if constexpr (!WIDE && DP == 16) {
      const u2 t = *reinterpret_cast<const u2 *>(at);
      f.v = u4{t[0], t[1], 0, 0};
    } else {
      f.v = *reinterpret_cast<const u4 *>(at);
    }
    return f;
  }
  static __device__ __forceinline__ void put_x(char *row, int kk, int g, int i, const RF &f) {
    char *at = row + ((SZ * d0(kk, g)) ^ x(i));
    if constexpr (!WIDE && DP == 16) *reinterpret_cast<u2 *>(at) = u2{f.v[0], f.v[1]};
    else *reinterpret_cast<u4 *>(at) = f.v;
  }
  // from global memory: dims past D and rows that are not there are zeros
  static __device__ __forceinline__ RF row_frag_of(const char *row, int kk, int g, int D, bool ok) {
    RF f;
    f.v = u4{0, 0, 0, 0};
    if (ok && d0(kk, g) < D) f = row_frag(row, kk, g);
    return f;
  }
  static __device__ __forceinline__ f4 dot(const RF &a, const RF &b, f4 c) {
    if constexpr (WIDE) {
#pragma unroll
      for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.v[j]), __uint_as_float(b.v[j]), c, 0, 0, 0);
      return c;
    } else if constexpr (DP == 16) {
      const u2 x = {a.v[0], a.v[1]}, y = {b.v[0], b.v[1]};
      if constexpr (TY == DI_F16)
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h4, x), __builtin_bit_cast(h4, y), c, 0, 0, 0);
      else
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, x), __builtin_bit_cast(s4, y), c, 0, 0, 0);
    } else if constexpr (TY == DI_F16) {
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a.v), __builtin_bit_cast(h8, b.v), c, 0, 0, 0);
    } else {
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a.v), __builtin_bit_cast(b8, b.v), c, 0, 0, 0);
    }
  }
  // columns 16 dt .. + 15 of the CH rows from row0 (a multiple of 16) of a TRS tile
  static __device__ __forceinline__ TF tr_frag(const char *tile, int stride, int row0, int dt, int i, int g) {
    TF f;
    if constexpr (WIDE) {
#pragma unroll
      for (int r = 0; r < 4; ++r) f.v[r] = *reinterpret_cast<const unsigned *>(tile + (row0 + 4 * g + r) * stride + 4 * (16 * dt + i));
    } else {
      const char *at = tile + (row0 + 4 * g + (i >> 2)) * stride + 32 * dt + ((8 * (i & 3)) ^ x(4 * g));
      const tr4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr4 __attribute__((address_space(3))) *)at);
      const tr4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr4 __attribute__((address_space(3))) *)(at + 16 * stride));
      const u2 a = __builtin_bit_cast(u2, lo), b = __builtin_bit_cast(u2, hi);
      f.v = u4{a[0], a[1], b[0], b[1]};
    }
    return f;
  }
  // result tiles (float32) -> operand of the contraction over their rows; 16-bit: rounded to nearest, half a step of the type -
  // the same relative error for every size of probability, and independent from one to the next in the sums that follow
  static __device__ __forceinline__ void pack(PF &f, int t, const f4 &p) {           // tile t of the operand
    if constexpr (WIDE) {
      f.v = __builtin_bit_cast(u4, p);
    } else {
      s4 s;
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] = TY == DI_F16 ? to_half_bits(p[r]) : to_bf_bits(p[r]);
      const u2 w = __builtin_bit_cast(u2, s);
      f.v[2 * t] = w[0];
      f.v[2 * t + 1] = w[1];
    }
  }
  static __device__ __forceinline__ f4 acc(const TF &a, const PF &p, f4 c) {
    if constexpr (WIDE) {
#pragma unroll
      for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.v[j]), __uint_as_float(p.v[j]), c, 0, 0, 0);
      return c;
    } else if constexpr (TY == DI_F16) {
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a.v), __builtin_bit_cast(h8, p.v), c, 0, 0, 0);
    } else {
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a.v), __builtin_bit_cast(b8, p.v), c, 0, 0, 0);
    }
  }
  // four consecutive head dims of an output row
  static __device__ __forceinline__ void store4(char *p, const f4 &x) {
    if constexpr (WIDE) {
      *reinterpret_cast<f4 *>(p) = x;
    } else {
      s4 s;
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] = TY == DI_F16 ? to_half_bits(x[r]) : to_bf_bits(x[r]);
      *reinterpret_cast<s4 *>(p) = s;
    }
  }
  static __device__ __forceinline__ float widen_dot(const RF &a, const RF &b) {      // products of the elements of two row fragments
    float t = 0.f;
    if constexpr (WIDE) {
#pragma unroll
      for (int j = 0; j < 4; ++j) t = fmaf(__uint_as_float(a.v[j]), __uint_as_float(b.v[j]), t);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const unsigned short x = (unsigned short)(a.v[j] >> (16 * e)), y = (unsigned short)(b.v[j] >> (16 * e));
          if constexpr (TY == DI_F16) t = fmaf((float)__builtin_bit_cast(_Float16, x), (float)__builtin_bit_cast(_Float16, y), t);
          else t = fmaf(__uint_as_float((unsigned)x << 16), __uint_as_float((unsigned)y << 16), t);
        }
      }
    }
    return t;
  }
};

// ---- attention dropout: keep or drop (row, key) from a counter-based hash, so that the backward regenerates the mask.  `mix` is
// the 32-bit integer mixer "lowbias32" (C. Wellons, "Prospecting for hash functions", 2018).  One 16-bit number per pair: the drop
// probability is a multiple of 2^-16, and the kept pairs are scaled by the reciprocal of exactly that.
__device__ __forceinline__ unsigned mix(unsigned x) {
  x ^= x >> 16; x *= 0x7feb352du;
  x ^= x >> 15; x *= 0x846ca68bu;
  return x ^ (x >> 16);
}
__device__ __forceinline__ unsigned drop_row(unsigned long long seed, unsigned long long row) {
  return mix(mix((unsigned)seed + (unsigned)row * 0x9e3779b9u) ^ (unsigned)(seed >> 32) ^ ((unsigned)(row >> 32) * 0x85ebca6bu));
}
// numbers of the keys 4 k4 .. 4 k4 + 3 of a row: low and high halves of two words
__device__ __forceinline__ unsigned drop_pair(unsigned row, unsigned k4, bool second) {
  const unsigned x = mix(row ^ (k4 * 0xc2b2ae35u));
  return second ? mix(x + 0x68bc21ebu) : x;
}

// n / d for 0 <= n < 2^31 by one multiplication (d fixed for the launch; T. Granlund and P. Montgomery, "Division by invariant integers
// using multiplication", 1994): with s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1,
// n / d = (mulhi(n, m) + n) >> s
struct Div {
  unsigned d, m, s;
  __host__ __device__ __forceinline__ unsigned of(unsigned n) const {
#ifdef __HIP_DEVICE_COMPILE__
    return (__umulhi(n, m) + n) >> s;
#else
    return (unsigned)((((unsigned long long)n * m >> 32) + n) >> s);
#endif
  }
};
inline Div div_by(unsigned d) {
  Div v = {d < 1 ? 1 : d, 0, 0};
  while ((1ull << v.s) < v.d) ++v.s;
  v.m = (unsigned)((((1ull << v.s) - v.d) << 32) / v.d + 1);
  return v;
}

struct Args {
  const char *q, *k, *v;
  char *o;                               // forward: (B, L, H D); backward: the forward's output
  const char *go;
  char *gq, *gk, *gv;
  float *lse, *delta;                    // (B Hk, G L); lse in the exp2 domain, -inf for an empty row
  float *part, *part_ml;                 // split over keys: sums (splits, B Hk, G L, D) and (max, sum) pairs
  float *part_k, *part_v;                // split over rows: (splits, B Hk, S, D)
  const int *klen;
  const unsigned char *kmask, *allowed;
  long long q_bs, q_rs, k_bs, k_rs, v_bs, v_rs, go_bs, go_rs, gk_bs, gk_rs, gv_bs, gv_rs, kmask_bs, allowed_bs, allowed_rs;   // strides (q .. gv: bytes)
  int B, L, S, Hk, G, D;
  int splits, range;                     // key (or row) ranges of a split grid
  int blocks;                            // row blocks (or key blocks)
  Div by_unit, by_blocks, by_hk, by_splits, by_L;              // unit = blocks * Hk
  int even;                              // blocks of the whole turns of 8 units
  bool ragged;                           // key lengths, few samples, more workgroups than CUs: blocks with keys first (where_ragged)
  Div by_walk, by_inner;                 // ragged: keys per step of a sample's blocks, blocks per step
  float scale2;                          // softmax scale * log2(e)
  float scale;
  unsigned drop;                         // threshold of 65536; 0 = no dropout
  float keep_scale;
  unsigned long long seed;
  const unsigned long long *seed_ptr;
};

__device__ __forceinline__ unsigned long long seed_of(const Args &a) { return a.seed + (a.seed_ptr != nullptr ? *a.seed_ptr : 0ull); }

// block -> (row block, key head, split, sample).  The blocks of one (sample, split) read the same memory rows - the same keys, or other
// heads of them - and go to one XCD, whose L2 they share; the (sample, split) units are dealt out to the XCDs in turn, so that samples
// of different lengths load them evenly.  Fewer than 8 units (or the last few): consecutive chunks of the block list per XCD.
struct Where {
  int blk, hk, sp, b;
};

__device__ __forceinline__ int keys_of(const Args &a, int b) {
  if (a.klen == nullptr) return a.S;
  const int n = a.klen[b];
  return n < 0 ? 0 : (n < a.S ? n : a.S);
}

// A row with a single key: its probability is 1 whatever the score, the score's gradient exactly 0 - not the rounding of dp - delta, all
// that would be left of gq and gk where every row is such a one.  Looked for where there are few keys at all.
constexpr int kFew = 16;
__device__ __forceinline__ bool one_key(const Args &a, int b, int query, int n) {
  int c = 0;
  for (int k = 0; k < n; ++k)
    c += (a.kmask == nullptr || a.kmask[b * a.kmask_bs + k] != 0) && (a.allowed == nullptr || a.allowed[b * a.allowed_bs + query * a.allowed_rs + k] != 0);
  return c <= 1;
}

// Samples of different lengths: the workgroups that have keys come first - dealt out to the XCDs as above, key blocks (equal work) in
// equal consecutive shares - and those without behind them.  Every wavefront finds its sample from the running sum of the samples' workgroups with keys (a lane each, so up
// to 64 samples).  A sample's workgroups are ordered by what its length cuts off: key ranges (row blocks), key blocks (KEYS).
// (4 x 511 x 4100, 2733, 1366, 0, four heads of 64 to a key head: gk and gv 121 -> 80 us, gq 54 -> 46, forward 41 -> 33; single
// queries of 16 samples with 0 .. 32 768 keys: 205 -> 196)
template <bool KEYS>
__device__ __forceinline__ Where where_ragged(const Args &a) {
  const int lane = threadIdx.x & 63, steps = KEYS ? a.blocks : a.splits, inner = (int)a.by_inner.d, all = steps * inner;
  int mine = 0;
  if (lane < a.B) mine = min(steps, (int)a.by_walk.of(keys_of(a, lane) + a.by_walk.d - 1)) * inner;
  int upto = mine;
#pragma unroll
  for (int x = 1; x < 64; x *= 2) {
    const int y = __shfl_up(upto, x);
    if (lane >= x) upto += y;
  }
  const int with = __builtin_amdgcn_readlane(upto, 63);
  int id = blockIdx.x, b;
  if (id < with) {
    if (KEYS) {
      id = xcd_remap(id, with);
    } else {                                                    // ranges of unequal length: whole units in turn, the last few in chunks
      const int even = (int)a.by_inner.of(with) / 8 * 8 * inner, xcd = id % 8, j = id / 8, turn = a.by_inner.of(j);
      id = id < even ? (turn * 8 + xcd) * inner + (j - turn * inner) : even + xcd_remap(id - even, with - even);
    }
    b = __builtin_popcountll(__ballot(upto <= id));            // samples that end before it (lanes behind the last one end at `with`)
    id -= __builtin_amdgcn_readlane(upto, b) - __builtin_amdgcn_readlane(mine, b);
  } else {
    id -= with;
    const int none = (lane + 1) * all - upto;
    b = __builtin_popcountll(__ballot(lane < a.B && none <= id));
    const int has = __builtin_amdgcn_readlane(mine, b);
    id += has - (__builtin_amdgcn_readlane(none, b) - (all - has));
  }
  Where w;
  w.b = b;
  if (KEYS) {
    w.blk = a.by_inner.of(id);
    const int at = id - w.blk * inner;
    w.sp = a.by_hk.of(at);
    w.hk = at - w.sp * a.Hk;
  } else {
    const int next = a.by_blocks.of(id);
    w.blk = id - next * a.blocks;
    w.sp = a.by_hk.of(next);
    w.hk = next - w.sp * a.Hk;
  }
  return w;
}

template <bool KEYS>
__device__ __forceinline__ Where where(const Args &a) {
  if (a.ragged) return where_ragged<KEYS>(a);
  const int unit = a.blocks * a.Hk;
  int id = blockIdx.x;
  if (id < a.even) {
    const int xcd = id % 8, j = id / 8, turn = a.by_unit.of(j);
    id = (turn * 8 + xcd) * unit + (j - turn * unit);
  } else {
    id = a.even + xcd_remap(id - a.even, gridDim.x - a.even);
  }
  Where w;
  int next = a.by_blocks.of(id);
  w.blk = id - next * a.blocks;
  id = next;
  next = a.by_hk.of(id);
  w.hk = id - next * a.Hk;
  id = next;
  w.b = a.by_splits.of(id);
  w.sp = id - w.b * a.splits;
  return w;
}

}  // namespace at
}  // namespace di
