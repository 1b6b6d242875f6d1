// Backward of LayerNorm with its residual add (layernorm.hip).  With h = (s - mu) rstd and g = gy w:
//
//     gs = rstd (g - mean_C(g) - h mean_C(g h)) (+ the gradient of the sum)      gx = gres = gs
//     gw = sum_rows gy h      gb = sum_rows gy
//
// ONE pass over the rows computes all four: s is formed again from x and res (the same bytes as a saved sum), the row's two
// means are one reduction, and a lane - which sees the same columns of every row its workgroup walks over - keeps its
// columns' shares of gw and gb in registers.  Every workgroup writes its shares as one record (float32), a second launch adds
// the records in a fixed order: the same bits on every run, no atomics.
//
// Bound by bytes: 72 000 x 128 (float32 stream, half-precision branch, 147 MB) 27 us = 5.4 TB/s, 8192 x 4096 bf16 with the sum's
// gradient (268 MB) 52 us = 5.1 TB/s; a 2 GB copy reaches 4.9 TB/s on this card.  Rows that are not 8 columns in steps of 16 bytes: 72 000 x 130
// float32 4.4 TB/s, 4096 x 4097 bf16 2.2 (2-byte accesses).  Above 8192 columns a row takes 1024 lanes of 128 registers, 22 - 96 of their values
// in scratch, and no next row is in flight: 1024 x 16 384 bf16 with the sum 63 us = 2.1 TB/s, 1024 x 12 000 float32 90 us = 2.2.
#include "layernorm.h"

namespace di {
namespace ln {

struct BwdArgs {
  const char *gy, *gsum, *x, *res, *w;
  const float *mean, *rstd;
  char *gx, *gres;
  float *part;                           // (gridDim.x, 2, C); a single workgroup writes gw and gb itself
  char *gw, *gb;
  long long rows, gy_rs, gsum_rs, x_rs, r_rs;   // row strides in BYTES
  int C, wsize, gx_size, gres_size;
  bool bf;
};

template <int LPR, int NV, bool VEC, int SX, int SR, int SY>
__global__ __launch_bounds__(threads_of(LPR)) void layernorm_bwd_kernel(BwdArgs a) {
  constexpr int T = threads_of(LPR), RPW = T / LPR;
  constexpr bool AHEAD = LPR < 1024;                            // 1024 threads have 128 registers each: no row in flight there
  __shared__ float red[LPR > 64 ? 4 * (LPR / 64) : 1];
  __shared__ float fold[RPW > 1 ? (RPW / 2) * LPR * NV * 16 : 1];
  const int l = threadIdx.x % LPR, C = a.C;
  const float inv = 1.f / (float)C;
  float w[NV][8], gw[NV][8], gb[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    load_param<LPR, VEC>(a.w, l, j, C, a.wsize, a.bf, w[j]);
#pragma unroll
    for (int e = 0; e < 8; ++e) gw[j][e] = gb[j][e] = 0.f;
  }
  Raw<SX, VEC> xr[NV], sr[NV];
  Raw<SR, VEC> rr[NV];
  Raw<SY, VEC> gr[NV];
  float mean = 0.f, rstd = 0.f;
  auto fetch = [&](long long row) {
    const char *px = a.x + row * a.x_rs, *pr = a.res + row * a.r_rs, *pg = a.gy + row * a.gy_rs;
#pragma unroll
    for (int j = 0; j < NV; ++j) load<LPR>(xr[j], px, l, j, C);
#pragma unroll
    for (int j = 0; j < NV; ++j) load<LPR>(gr[j], pg, l, j, C);
    if (a.res != nullptr) {
#pragma unroll
      for (int j = 0; j < NV; ++j) load<LPR>(rr[j], pr, l, j, C);
    }
    mean = a.mean[row];
    rstd = a.rstd[row];
  };
  const long long step = (long long)gridDim.x * RPW, first = (long long)blockIdx.x * RPW + threadIdx.x / LPR;
  int flip = 0;
  if (AHEAD && first < a.rows) fetch(first);
  for (long long row = first; row < a.rows; row += step) {      // LPR > 64: one trip count per workgroup (RPW = 1)
    float h[NV][8], g[NV][8];
    if (!AHEAD) fetch(row);
    const float mu = mean, rs = rstd;
    if (a.gsum != nullptr) {                                    // needed last: in flight behind the reduction
      const char *ps = a.gsum + row * a.gsum_rs;
#pragma unroll
      for (int j = 0; j < NV; ++j) load<LPR>(sr[j], ps, l, j, C);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      unpack(xr[j], a.bf, h[j]);
      unpack(gr[j], a.bf, g[j]);
    }
    if (a.res != nullptr) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float r[8];
        unpack(rr[j], a.bf, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[j][e] += r[e];
      }
    }
    if (AHEAD && row + step < a.rows) fetch(row + step);
    float t[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[j][e] = (h[j][e] - mu) * rs;                          // columns past C: g = 0, so their h reaches no sum
        gw[j][e] = fmaf(g[j][e], h[j][e], gw[j][e]);
        gb[j][e] += g[j][e];
        g[j][e] *= w[j][e];
        t[0] += g[j][e];
        t[1] = fmaf(g[j][e], h[j][e], t[1]);
      }
    row_sum<LPR, 2>(t, red, flip);
    const float m0 = t[0] * inv, m1 = t[1] * inv;
    char *px = a.gx + row * C * a.gx_size, *pr = a.gres + row * C * a.gres_size;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) g[j][e] = rs * (g[j][e] - m0 - h[j][e] * m1);
      if (a.gsum != nullptr) {
        float add[8];
        unpack(sr[j], a.bf, add);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[j][e] += add[e];
      }
      store<LPR, VEC>(px, l, j, C, a.gx_size, a.bf, g[j]);
      if (a.gres != nullptr) store<LPR, VEC>(pr, l, j, C, a.gres_size, a.bf, g[j]);
    }
  }
  // the workgroup's RPW row groups hold the same columns: fold them by halves
  if constexpr (RPW > 1) {
    const int rg = threadIdx.x / LPR;
#pragma unroll
    for (int n = RPW / 2; n >= 1; n >>= 1) {
      __syncthreads();
      if (rg >= n && rg < 2 * n) {
        float *at = fold + (rg - n) * (LPR * NV * 16) + l;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            at[(16 * j + e) * LPR] = gw[j][e];
            at[(16 * j + 8 + e) * LPR] = gb[j][e];
          }
      }
      __syncthreads();
      if (rg < n) {
        const float *at = fold + rg * (LPR * NV * 16) + l;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            gw[j][e] += at[(16 * j + e) * LPR];
            gb[j][e] += at[(16 * j + 8 + e) * LPR];
          }
      }
    }
  }
  if (threadIdx.x < LPR && gridDim.x == 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      store<LPR, VEC>(a.gw, l, j, C, a.wsize, a.bf, gw[j]);
      store<LPR, VEC>(a.gb, l, j, C, a.wsize, a.bf, gb[j]);
    }
  } else if (threadIdx.x < LPR) {
    char *rec = reinterpret_cast<char *>(a.part + (size_t)blockIdx.x * 2 * C);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      store<LPR, VEC>(rec, l, j, C, 4, false, gw[j]);
      store<LPR, VEC>(rec + 4 * (size_t)C, l, j, C, 4, false, gb[j]);
    }
  }
}

// gw | gb = the sum of the G records: 16 columns x 64 slices of the records per workgroup.  (1024 records of
// 256 columns: 6.6 us with 16 slices, whose loads follow each other, 3.9 us with 64; 512 records of 8192 columns: 6.6 us with both)
__global__ __launch_bounds__(1024) void layernorm_param_kernel(const float *__restrict__ part, int G, int C, char *__restrict__ gw,
                                                               char *__restrict__ gb, int size, bool bf) {
  __shared__ float s[64][17];
  const int i = threadIdx.x & 15, k = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + i, n = 2 * C;
  float t = 0.f;
  if (c < n) {
    int r = k;
    float u0 = 0.f, u1 = 0.f, u2 = 0.f, u3 = 0.f;               // four loads in flight
    for (; r + 192 < G; r += 256) {
      u0 += part[(size_t)r * n + c];
      u1 += part[(size_t)(r + 64) * n + c];
      u2 += part[(size_t)(r + 128) * n + c];
      u3 += part[(size_t)(r + 192) * n + c];
    }
    for (; r < G; r += 64) u0 += part[(size_t)r * n + c];
    t = (u0 + u1) + (u2 + u3);
  }
  s[k][i] = t;
  __syncthreads();
  if (k < 4) {                                                  // one wavefront: 16 columns x 4 quarters of the slices
    float u = 0.f;
#pragma unroll
    for (int q = 0; q < 16; ++q) u += s[16 * k + q][i];
    u += __shfl_xor(u, 16);
    u += __shfl_xor(u, 32);
    if (k == 0 && c < n) {
      char *dst = c < C ? gw : gb;
      const int at = c < C ? c : c - C;
      if (size == 2) reinterpret_cast<unsigned short *>(dst)[at] = narrow(u, bf);
      else reinterpret_cast<float *>(dst)[at] = u;
    }
  }
}

// Up to this many passes one workgroup walks over all rows and the second launch falls away (200 x 128, 13 passes: 11.3 us in one
// workgroup, 4.4 + 2.3 in 13 and the reduction: a pass costs 0.8 us, the reduction's launch 2 - 3)
constexpr int kOnePass = 3;

// records = workgroups of the pass over the rows
static int records(long long rows, int C) {
  const int cus = device_cus();
  if (cus <= 0) return -1;
#define DI_LN_G(LPR, NV, V)                                                                                                \
  do {                                                                                                                     \
    constexpr int RPW = threads_of(LPR) / LPR;                                                                             \
    const long long passes = (rows + RPW - 1) / RPW, most = (long long)cus * (LPR <= 64 ? 4 : 2);                          \
    return passes <= kOnePass ? (passes > 0) : (int)(passes < most ? passes : most);                                       \
  } while (0)
  DI_LN_CONFIGS(DI_LN_G, true);
#undef DI_LN_G
}

template <int SX, int SR, int SY>
static int launch(const BwdArgs &a, bool vec, int G, hipStream_t s) {
  const int C = a.C;
#define DI_LN_GO(LPR, NV, V)                                                                                               \
  hipLaunchKernelGGL((layernorm_bwd_kernel<LPR, NV, V, SX, SR, SY>), dim3((unsigned)G), dim3(threads_of(LPR)), 0, s, a)
  if (vec) DI_LN_CONFIGS(DI_LN_GO, true);
  else DI_LN_CONFIGS(DI_LN_GO, false);
#undef DI_LN_GO
  return check_launch("layernorm_bwd");
}

}  // namespace ln
}  // namespace di

extern "C" {

long long di_layernorm_bwd_workspace_floats(long long rows, int C) {
  if (rows < 0 || C <= 0 || C > di::ln::kMaxC) return -1;
  const int G = di::ln::records(rows, C);
  return G < 0 ? -1 : (long long)G * 2 * C;
}

int di_layernorm_bwd(const void *gy, long long gy_row_stride, int y_dtype, const void *gsum, long long gsum_row_stride, const void *x,
                     long long x_row_stride, int x_dtype, const void *res, long long res_row_stride, int res_dtype, const void *weight,
                     int w_dtype, const float *mean, const float *rstd, void *gx, int gx_dtype, void *gres, void *gweight, void *gbias,
                     float *workspace, long long rows, int C, void *stream) {
  using namespace di::ln;
  DI_REQUIRE(rows >= 0 && C > 0 && C <= kMaxC, "layernorm_bwd: %d columns (1 .. %d are supported)", C, kMaxC);
  DI_REQUIRE(known(x_dtype) && known(w_dtype) && known(y_dtype) && known(gx_dtype) && (res == nullptr || known(res_dtype)),
             "layernorm_bwd: unsupported dtype");
  if (res == nullptr) res_dtype = x_dtype;
  const int types[5] = {x_dtype, res_dtype, w_dtype, y_dtype, gx_dtype};
  const int bf = half_type(types, 5);
  DI_REQUIRE(bf >= 0, "layernorm_bwd: float16 and bfloat16 in one call");
  const int sx = size_of(x_dtype), sr = size_of(res_dtype), sy = size_of(y_dtype), sw = size_of(w_dtype), sg = size_of(gx_dtype);
  DI_REQUIRE(sy == 4 || (sx == 2 && sr == 2), "layernorm_bwd: a 16-bit output of a float32 input");
  DI_REQUIRE(gres == nullptr || res != nullptr, "layernorm_bwd: a gradient for a residual that is not there");
  DI_REQUIRE(gweight && gbias, "layernorm_bwd: null pointer");
  hipStream_t s = (hipStream_t)stream;
  int G = 0;
  if (rows > 0) {
    DI_REQUIRE(gy && x && weight && mean && rstd && gx && workspace, "layernorm_bwd: null pointer");
    G = records(rows, C);
    if (G < 0) return DI_ERR_LAUNCH;
    const bool vec = C % 8 == 0 && aligned16(gy, gy_row_stride, sy) && aligned16(gsum, gsum_row_stride, sx) &&
                     aligned16(x, x_row_stride, sx) && aligned16(res, res_row_stride, sr) && aligned16(weight, 0, sw) &&
                     aligned16(gx, C, sg) && aligned16(gres, C, sr) && aligned16(workspace, C, 4) && aligned16(gweight, 0, sw) && aligned16(gbias, 0, sw);
    const BwdArgs a = {(const char *)gy, (const char *)gsum, (const char *)x, (const char *)res, (const char *)weight, mean, rstd,
                       (char *)gx, (char *)gres, workspace, (char *)gweight, (char *)gbias, rows, gy_row_stride * sy, gsum_row_stride * sx, x_row_stride * sx,
                       res_row_stride * sr, C, sw, sg, sr, bf == 1};
    int rc;
    if (sx == 2) {
      if (sr == 4) rc = launch<2, 4, 4>(a, vec, G, s);
      else rc = sy == 2 ? launch<2, 2, 2>(a, vec, G, s) : launch<2, 2, 4>(a, vec, G, s);
    } else {
      rc = sr == 2 ? launch<4, 2, 4>(a, vec, G, s) : launch<4, 4, 4>(a, vec, G, s);
    }
    if (rc != DI_OK || G == 1) return rc;
  }
  hipLaunchKernelGGL(layernorm_param_kernel, dim3((2 * C + 15) / 16), dim3(1024), 0, s, workspace, G, C, (char *)gweight, (char *)gbias,
                     sw, bf == 1);
  return di::check_launch("layernorm_bwd");
}

}  // extern "C"
