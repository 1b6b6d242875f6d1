// LayerNorm with its residual add, any width to 16 384, forward (inference and training form); the backward is in
// layernorm_bwd.hip.  Reference: every post-norm step `norm(x + dropout(branch))` of decoder_utils.py:96-113, :743-756,
// :824-837 and of the ++ neck's layers, and the Swin backbone's norms (swin.py).
//
//     s = x (+ res)      mu = mean_C(s)      rstd = (mean_C((s - mu)^2) + eps)^-1/2      y = (s - mu) rstd w + b
//
// Eight operations an element: bound by the bytes of x, res, y (and s).  Workgroups walk over the rows with the next row's
// loads in flight while the current one is reduced; weight and bias stay in registers.  72 000 x 128 (float32 stream, half-
// precision branch, 92 MB): 18 us = 5.1 TB/s; 8192 x 4096 bf16 with the sum (268 MB): 47 us = 5.7 TB/s.  When the sum is asked for it is
// rounded to its type first and what is normalised is that rounded value: the network carries it on, and the backward reads it.
#include "layernorm.h"

namespace di {
namespace ln {

struct FwdArgs {
  const char *x, *res, *w, *b;
  char *y, *sum;
  float *mean, *rstd;
  long long rows, x_rs, r_rs;            // row strides in BYTES
  int C, wsize;
  float eps;
  bool bf;
};

template <int LPR, int NV, bool VEC, int SX, int SR, int SY>
__global__ __launch_bounds__(threads_of(LPR)) void layernorm_fwd_kernel(FwdArgs a) {
  constexpr int RPW = threads_of(LPR) / LPR;                    // rows per workgroup and pass
  __shared__ float red[LPR > 64 ? 2 * (LPR / 64) : 1];
  const int l = threadIdx.x % LPR, C = a.C;
  const float inv = 1.f / (float)C;
  float w[NV][8], b[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    load_param<LPR, VEC>(a.w, l, j, C, a.wsize, a.bf, w[j]);
    load_param<LPR, VEC>(a.b, l, j, C, a.wsize, a.bf, b[j]);
  }
  Raw<SX, VEC> xr[NV];
  Raw<SR, VEC> rr[NV];
  auto fetch = [&](long long row) {
    const char *px = a.x + row * a.x_rs, *pr = a.res + row * a.r_rs;
#pragma unroll
    for (int j = 0; j < NV; ++j) load<LPR>(xr[j], px, l, j, C);
    if (a.res != nullptr) {
#pragma unroll
      for (int j = 0; j < NV; ++j) load<LPR>(rr[j], pr, l, j, C);
    }
  };
  const long long step = (long long)gridDim.x * RPW, first = (long long)blockIdx.x * RPW + threadIdx.x / LPR;
  // LPR > 64: the trip count is the same for the whole workgroup (RPW = 1), as the barriers of row_sum need
  int flip = 0;
  if (first < a.rows) fetch(first);
  for (long long row = first; row < a.rows; row += step) {
    float s[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) unpack(xr[j], a.bf, s[j]);
    if (a.res != nullptr) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float r[8];
        unpack(rr[j], a.bf, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[j][e] += r[e];
      }
    }
    if (row + step < a.rows) fetch(row + step);
    if (a.sum != nullptr) {
      char *ps = a.sum + row * C * SX;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (SX == 2) {
#pragma unroll
          for (int e = 0; e < 8; ++e) s[j][e] = widen(narrow(s[j][e], a.bf), a.bf);
        }
        store<LPR, VEC>(ps, l, j, C, SX, a.bf, s[j]);
      }
    }
    float t[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) t[0] += s[j][e];              // columns past C hold zeros
    row_sum<LPR, 1>(t, red, flip);
    const float mean = t[0] * inv;
    t[0] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[j][e] = column_ok<LPR, VEC>(l, j, e, C) ? s[j][e] - mean : 0.f;
        t[0] = fmaf(s[j][e], s[j][e], t[0]);
      }
    row_sum<LPR, 1>(t, red, flip);
    const float rstd = 1.f / sqrtf(t[0] * inv + a.eps);
    if (a.mean != nullptr && l == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    char *py = a.y + row * C * SY;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s[j][e] = fmaf(s[j][e] * rstd, w[j][e], b[j][e]);
      store<LPR, VEC>(py, l, j, C, SY, a.bf, s[j]);
    }
  }
}

template <int SX, int SR, int SY>
static int launch(const FwdArgs &a, bool vec, hipStream_t s) {
  const int C = a.C;
  const int cus = device_cus();
  if (cus <= 0) return DI_ERR_LAUNCH;
#define DI_LN_GO(LPR, NV, V)                                                                                               \
  do {                                                                                                                     \
    constexpr int RPW = threads_of(LPR) / LPR;                                                                             \
    const long long passes = (a.rows + RPW - 1) / RPW, most = (long long)cus * (2048 / threads_of(LPR));                   \
    hipLaunchKernelGGL((layernorm_fwd_kernel<LPR, NV, V, SX, SR, SY>), dim3((unsigned)(passes < most ? passes : most)),    \
                       dim3(threads_of(LPR)), 0, s, a);                                                                    \
  } while (0)
  if (vec) DI_LN_CONFIGS(DI_LN_GO, true);
  else DI_LN_CONFIGS(DI_LN_GO, false);
#undef DI_LN_GO
  return check_launch("layernorm_fwd");
}

}  // namespace ln
}  // namespace di

extern "C" int di_layernorm_fwd(const void *x, long long x_row_stride, int x_dtype, const void *res, long long res_row_stride,
                                int res_dtype, const void *weight, const void *bias, int w_dtype, void *y, int y_dtype, void *sum,
                                float *mean, float *rstd, long long rows, int C, float eps, void *stream) {
  using namespace di::ln;
  DI_REQUIRE(rows >= 0 && C > 0 && C <= kMaxC, "layernorm: %d columns (1 .. %d are supported)", C, kMaxC);
  DI_REQUIRE(known(x_dtype) && known(w_dtype) && known(y_dtype) && (res == nullptr || known(res_dtype)), "layernorm: unsupported dtype");
  if (res == nullptr) res_dtype = x_dtype;
  const int types[4] = {x_dtype, res_dtype, w_dtype, y_dtype};
  const int bf = half_type(types, 4);
  DI_REQUIRE(bf >= 0, "layernorm: float16 and bfloat16 in one call");
  const int sx = size_of(x_dtype), sr = size_of(res_dtype), sy = size_of(y_dtype), sw = size_of(w_dtype);
  DI_REQUIRE(sy == 4 || (sx == 2 && sr == 2), "layernorm: a 16-bit output of a float32 input");
  DI_REQUIRE((mean == nullptr) == (rstd == nullptr), "layernorm: mean and rstd go together");
  if (rows == 0) return DI_OK;
  DI_REQUIRE(x && weight && bias && y, "layernorm: null pointer");
  const bool vec = C % 8 == 0 && aligned16(x, x_row_stride, sx) && aligned16(res, res_row_stride, sr) && aligned16(weight, 0, sw) &&
                   aligned16(bias, 0, sw) && aligned16(y, C, sy) && aligned16(sum, C, sx);
  const FwdArgs a = {(const char *)x, (const char *)res, (const char *)weight, (const char *)bias, (char *)y, (char *)sum, mean, rstd,
                     rows, x_row_stride * sx, res == nullptr ? 0 : res_row_stride * sr, C, sw, eps, bf == 1};
  hipStream_t s = (hipStream_t)stream;
  if (sx == 2) {
    if (sr == 4) return launch<2, 4, 4>(a, vec, s);
    return sy == 2 ? launch<2, 2, 2>(a, vec, s) : launch<2, 2, 4>(a, vec, s);
  }
  return sr == 2 ? launch<4, 2, 4>(a, vec, s) : launch<4, 4, 4>(a, vec, s);
}
