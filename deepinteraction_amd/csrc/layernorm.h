// Row layout and typed row access shared by the LayerNorm kernels (layernorm.hip, layernorm_bwd.hip).
//
// A row of C elements belongs to LPR lanes (16 = a DPP row, 64 = a wavefront, 256 - 1024 = a workgroup) that hold it in
// registers as NV chunks of 8: the statistics are taken from registers (mean first, then the centred squares, float32), so a
// row is read once.  VEC: chunk j of lane l is the columns 8 (l + LPR j) .. + 7, one or two 16-byte accesses; otherwise
// (C % 8 != 0, or a row that does not start on 16 bytes) element e of chunk j is column l + LPR (8 j + e), 2- or 4-byte
// accesses that are contiguous over the lanes.
#pragma once
#include "di_common.h"

namespace di {
namespace ln {

typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

template <int SZ, bool VEC>
struct Raw;
template <>
struct Raw<2, true> { u4 v; };
template <>
struct Raw<4, true> { u4 v, w; };
template <>
struct Raw<2, false> { unsigned short e[8]; };
template <>
struct Raw<4, false> { float e[8]; };

__device__ __forceinline__ float widen(unsigned short u, bool bf) {
  return bf ? __uint_as_float((unsigned)u << 16) : (float)__builtin_bit_cast(_Float16, u);
}
__device__ __forceinline__ unsigned short narrow(float f, bool bf) {          // round to nearest even: half a step of the type
  return bf ? __builtin_bit_cast(unsigned short, (__bf16)f) : __builtin_bit_cast(unsigned short, (_Float16)f);
}

// `row` = first byte of the row, `j` the chunk
template <int LPR>
__device__ __forceinline__ void load(Raw<2, true> &r, const char *row, int l, int j, int C) {
  const int c = 8 * (l + LPR * j);
  r.v = c < C ? *reinterpret_cast<const u4 *>(row + 2 * c) : u4{0, 0, 0, 0};
}
template <int LPR>
__device__ __forceinline__ void load(Raw<4, true> &r, const char *row, int l, int j, int C) {
  const int c = 8 * (l + LPR * j);
  r.v = r.w = u4{0, 0, 0, 0};
  if (c < C) {
    r.v = *reinterpret_cast<const u4 *>(row + 4 * c);
    r.w = *reinterpret_cast<const u4 *>(row + 4 * c + 16);
  }
}
template <int LPR>
__device__ __forceinline__ void load(Raw<2, false> &r, const char *row, int l, int j, int C) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = l + LPR * (8 * j + e);
    r.e[e] = c < C ? reinterpret_cast<const unsigned short *>(row)[c] : 0;
  }
}
template <int LPR>
__device__ __forceinline__ void load(Raw<4, false> &r, const char *row, int l, int j, int C) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = l + LPR * (8 * j + e);
    r.e[e] = c < C ? reinterpret_cast<const float *>(row)[c] : 0.f;
  }
}

template <bool VEC>
__device__ __forceinline__ void unpack(const Raw<2, VEC> &r, bool bf, float (&f)[8]) {
  if constexpr (VEC) {
    const unsigned w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = widen((unsigned short)(w[i] & 0xffffu), bf);
      f[2 * i + 1] = widen((unsigned short)(w[i] >> 16), bf);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = widen(r.e[i], bf);
  }
}
template <bool VEC>
__device__ __forceinline__ void unpack(const Raw<4, VEC> &r, bool, float (&f)[8]) {
  if constexpr (VEC) {
    const unsigned w[8] = {r.v.x, r.v.y, r.v.z, r.v.w, r.w.x, r.w.y, r.w.z, r.w.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = r.e[i];
  }
}

// store chunk j; `size` 2 or 4 (uniform over the launch)
template <int LPR, bool VEC>
__device__ __forceinline__ void store(char *row, int l, int j, int C, int size, bool bf, const float (&f)[8]) {
  if constexpr (VEC) {
    const int c = 8 * (l + LPR * j);
    if (c >= C) return;
    if (size == 2) {
      unsigned w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (unsigned)narrow(f[2 * i], bf) | ((unsigned)narrow(f[2 * i + 1], bf) << 16);
      *reinterpret_cast<u4 *>(row + 2 * c) = u4{w[0], w[1], w[2], w[3]};
    } else {
      *reinterpret_cast<f4 *>(row + 4 * c) = f4{f[0], f[1], f[2], f[3]};
      *reinterpret_cast<f4 *>(row + 4 * c + 16) = f4{f[4], f[5], f[6], f[7]};
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = l + LPR * (8 * j + e);
      if (c < C) {
        if (size == 2) reinterpret_cast<unsigned short *>(row)[c] = narrow(f[e], bf);
        else reinterpret_cast<float *>(row)[c] = f[e];
      }
    }
  }
}

// the weight's or bias's chunk j (float32 or the call's 16-bit type)
template <int LPR, bool VEC>
__device__ __forceinline__ void load_param(const char *p, int l, int j, int C, int size, bool bf, float (&f)[8]) {
  if (size == 2) {
    Raw<2, VEC> r;
    load<LPR>(r, p, l, j, C);
    unpack(r, bf, f);
  } else {
    Raw<4, VEC> r;
    load<LPR>(r, p, l, j, C);
    unpack(r, bf, f);
  }
}

template <int LPR, bool VEC>
__device__ __forceinline__ bool column_ok(int l, int j, int e, int C) {
  return VEC ? 8 * (l + LPR * j) < C : l + LPR * (8 * j + e) < C;
}

// The row's sums of N values: every lane of the row's LPR lanes ends with them.  `red`: LDS of 2 N (LPR / 64) floats, its
// halves used in turn (`flip`) so that one barrier per call is enough: a wavefront can write a half again only after every
// wavefront has passed the barrier of the call in between, which is after its reads of that half.
template <int LPR, int N>
__device__ __forceinline__ void row_sum(float (&s)[N], float *red, int &flip) {
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = row16_sum(s[i]);
  if constexpr (LPR >= 64) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s[i] += __shfl_xor(s[i], 16);
      s[i] += __shfl_xor(s[i], 32);
    }
  }
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    float *at = red + flip * (N * W);
    flip ^= 1;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) at[i * W + wave] = s[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) t += at[i * W + w];
      s[i] = t;
    }
  }
}

constexpr int threads_of(int LPR) { return LPR > 256 ? LPR : 256; }

// host: the lanes and chunks for a row of C elements
#define DI_LN_CONFIGS(DO, ...)                                                                                             \
  do {                                                                                                                     \
    if (C <= 128) DO(16, 1, __VA_ARGS__);                                                                                  \
    else if (C <= 512) DO(64, 1, __VA_ARGS__);                                                                             \
    else if (C <= 1024) DO(64, 2, __VA_ARGS__);                                                                            \
    else if (C <= 2048) DO(256, 1, __VA_ARGS__);                                                                           \
    else if (C <= 4096) DO(256, 2, __VA_ARGS__);                                                                           \
    else if (C <= 8192) DO(512, 2, __VA_ARGS__);                                                                           \
    else DO(1024, 2, __VA_ARGS__);                                                                                         \
  } while (0)

constexpr int kMaxC = 16384;

inline int size_of(int dtype) { return dtype == DI_F32 ? 4 : 2; }
inline bool known(int dtype) { return dtype == DI_F32 || dtype == DI_F16 || dtype == DI_BF16; }
inline bool aligned16(const void *p, long long row_stride, int size) {
  return p == nullptr || (((uintptr_t)p & 15) == 0 && (row_stride * size) % 16 == 0);
}
// one 16-bit type per call: -1 when two differ, else whether it is bf16
inline int half_type(const int *dtypes, int n) {
  int t = 0;
  for (int i = 0; i < n; ++i)
    if (dtypes[i] != DI_F32) {
      if (t != 0 && t != dtypes[i]) return -1;
      t = dtypes[i];
    }
  return t == DI_BF16;
}

}  // namespace ln
}  // namespace di
