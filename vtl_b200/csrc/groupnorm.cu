// Group norm with an activation, channels last: x[B, S, C] (S positions: H * W of a feature map, the length of a
// sequence, 1 for plain features), C channels in `groups` equal groups.  Per sample and group, over S * C/groups values,
//   h = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps) (biased variance),  z = gamma_c * h + beta_c,  y = act(z).
// Backward, with dz = g * act'(z) and n = S * C/groups:
//   dgamma_c = sum over samples and positions of dz * h,   dbeta_c = sum of dz,
//   dx = rstd * (gamma_c * dz - (sum gamma dz) / n - h * (sum gamma dz h) / n), the sums over the group.
#include "common.cuh"

namespace {

struct GnDims {
  int B, S, C, G, width;  // width = C / G
};

template <int ACT>
__device__ __forceinline__ float act(float z) {
  if (ACT == VTLB_ACT_RELU) return z < 0.0f ? 0.0f : z;
  if (ACT == VTLB_ACT_SILU) return z / (1.0f + expf(-z));
  return z;
}

// g * act'(z).  ReLU passes the gradient at exactly zero (nn/internal/activation.v:78-87).  z close to zero is
// evaluated again in f64: rounding must not decide which side it is on.
template <int ACT>
__device__ __forceinline__ float act_bwd(float g, float x, float mean, float rstd, float gamma, float beta, float h) {
  if (ACT == VTLB_ACT_NONE) return g;
  const float a = __fmul_rn(gamma, h), z = __fadd_rn(a, beta);
  if (ACT == VTLB_ACT_RELU) {
    if (fabsf(z) <= 1e-6f * (fabsf(a) + fabsf(beta))) {
      const double zd = ((double)x - (double)mean) * (double)rstd * (double)gamma + (double)beta;
      return zd < 0.0 ? 0.0f : g;
    }
    return z < 0.0f ? 0.0f : g;
  }
  const float s = 1.0f / (1.0f + expf(-z));
  return g * (s * (1.0f + z * (1.0f - s)));
}

constexpr int kRows = 256;  // rows of x per CTA of the sums below

// Sums of one column of [chunk of rows] in f64 into partial[b][chunk][c]: of x and x^2 (forward), of dz and dz * h.
template <int ACT, bool BWD>
__global__ void __launch_bounds__(256) gn_sums_kernel(const float* x, const float* g, const float* gamma,
                                                      const float* beta, const float* mean, const float* rstd, GnDims d,
                                                      double2* partial) {
  __shared__ double2 sm[8][32];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cl, chunk = blockIdx.y, b = blockIdx.z;
  const int r1 = min(d.S, (chunk + 1) * kRows);
  double2 acc = make_double2(0.0, 0.0);
  if (c < d.C) {
    float mu = 0.f, rs = 0.f, ga = 1.f, be = 0.f;
    if (BWD) {
      mu = mean[b * d.G + c / d.width], rs = rstd[b * d.G + c / d.width];
      if (gamma) ga = gamma[c];
      if (beta) be = beta[c];
    }
    for (int r = chunk * kRows + rl; r < r1; r += 8) {
      const size_t i = ((size_t)b * d.S + r) * d.C + c;
      const float v = x[i];
      if (BWD) {
        const float h = __fmul_rn(__fsub_rn(v, mu), rs), dz = act_bwd<ACT>(g[i], v, mu, rs, ga, be, h);
        acc.x += (double)dz;
        acc.y += (double)dz * (double)h;
      } else {
        acc.x += (double)v;
        acc.y += (double)v * (double)v;
      }
    }
  }
  sm[rl][cl] = acc;
  __syncthreads();
  if (rl == 0 && c < d.C) {
    for (int k = 1; k < 8; ++k) acc.x += sm[k][cl].x, acc.y += sm[k][cl].y;
    partial[((size_t)b * gridDim.y + chunk) * d.C + c] = acc;
  }
}

// One warp per (sample, group): the sums over chunks and channels, in a fixed order.
template <bool BWD>
__global__ void __launch_bounds__(256) gn_groups_kernel(const double2* partial, int chunks, GnDims d, const float* gamma,
                                                        double eps, float* mean, float* rstd, float2* coef) {
  const int lane = threadIdx.x & 31;
  const size_t k = (blockIdx.x * (size_t)blockDim.x + threadIdx.x) >> 5;
  if (k >= (size_t)d.B * d.G) return;
  const int b = (int)(k / d.G), grp = (int)(k % d.G);
  double s0 = 0.0, s1 = 0.0;
  for (int i = lane; i < chunks * d.width; i += 32) {
    const int c = grp * d.width + i % d.width;
    const double2 p = partial[((size_t)b * chunks + i / d.width) * d.C + c];
    const double w = BWD && gamma ? (double)gamma[c] : 1.0;
    s0 += w * p.x, s1 += w * p.y;
  }
  for (int o = 16; o; o >>= 1) s0 += __shfl_xor_sync(~0u, s0, o), s1 += __shfl_xor_sync(~0u, s1, o);
  if (lane) return;
  const double n = (double)d.S * d.width;
  if (BWD) {
    coef[k] = make_float2((float)(s0 / n), (float)(s1 / n));
  } else {
    const double mu = s0 / n, var = s1 / n - mu * mu;
    mean[k] = (float)mu;
    rstd[k] = (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + eps));
  }
}

// dgamma and dbeta: one thread per channel sums over samples and chunks.
__global__ void __launch_bounds__(64) gn_params_kernel(const double2* partial, int rows, int C, float* dgamma, float* dbeta) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= C) return;
  double s0 = 0.0, s1 = 0.0;
  for (int r = 0; r < rows; ++r) s0 += partial[(size_t)r * C + c].x, s1 += partial[(size_t)r * C + c].y;
  if (dbeta) dbeta[c] = (float)s0;
  if (dgamma) dgamma[c] = (float)s1;
}

template <int ACT, bool BWD>
__global__ void __launch_bounds__(256) gn_apply_kernel(const float* x, const float* g, const float* gamma,
                                                       const float* beta, const float* mean, const float* rstd,
                                                       const float2* coef, GnDims d, float* out) {
  const size_t total = (size_t)d.B * d.S * d.C;
  for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
    const int c = (int)(i % d.C);
    const size_t k = i / ((size_t)d.S * d.C) * d.G + c / d.width;
    const float mu = mean[k], rs = rstd[k], ga = gamma ? gamma[c] : 1.0f, be = beta ? beta[c] : 0.0f, v = x[i];
    const float h = __fmul_rn(__fsub_rn(v, mu), rs);
    if (BWD) {
      const float dz = act_bwd<ACT>(g[i], v, mu, rs, ga, be, h);
      const float2 cf = coef[k];
      out[i] = rs * (ga * dz - cf.x - h * cf.y);
    } else {
      out[i] = act<ACT>(ga * h + be);
    }
  }
}

int check_dims(vtlb_ctx* ctx, const char* fn, int B, int S, int C, int groups, int act_kind, GnDims* d) {
  if (B <= 0 || S <= 0 || C <= 0 || groups <= 0 || C % groups)
    return vtlb_fail(ctx, VTLB_EINVAL, "%s: bad shape B=%d S=%d C=%d groups=%d", fn, B, S, C, groups);
  if (act_kind != VTLB_ACT_NONE && act_kind != VTLB_ACT_RELU && act_kind != VTLB_ACT_SILU)
    return vtlb_fail(ctx, VTLB_EINVAL, "%s: unknown activation %d", fn, act_kind);
  if (B > 65535 || S > 65535 * kRows)
    return vtlb_fail(ctx, VTLB_EINVAL, "%s: B=%d S=%d is beyond 65535 samples of %d positions", fn, B, S, 65535 * kRows);
  *d = GnDims{B, S, C, groups, C / groups};
  return VTLB_OK;
}

template <int ACT>
int gn_forward(vtlb_ctx* ctx, const float* x, GnDims d, const float* gamma, const float* beta, double eps, float* y,
               float* mean, float* rstd) {
  const int chunks = (d.S + kRows - 1) / kRows;
  vtlb_workspace ws(ctx);
  void* partial = nullptr;
  if (int rc = ws.get((size_t)d.B * chunks * d.C * sizeof(double2), &partial)) return rc;
  gn_sums_kernel<ACT, false><<<dim3((d.C + 31) / 32, chunks, d.B), 256, 0, ctx->stream>>>(
      x, nullptr, nullptr, nullptr, nullptr, nullptr, d, (double2*)partial);
  VTLB_LAUNCHED(ctx);
  gn_groups_kernel<false><<<(unsigned)(((size_t)d.B * d.G + 7) / 8), 256, 0, ctx->stream>>>(
      (const double2*)partial, chunks, d, nullptr, eps, mean, rstd, nullptr);
  VTLB_LAUNCHED(ctx);
  gn_apply_kernel<ACT, false><<<ctx->sm_count * 8, 256, 0, ctx->stream>>>(x, nullptr, gamma, beta, mean, rstd, nullptr, d, y);
  VTLB_LAUNCHED(ctx);
  return VTLB_OK;
}

template <int ACT>
int gn_backward(vtlb_ctx* ctx, const float* g, const float* x, GnDims d, const float* gamma, const float* beta,
                const float* mean, const float* rstd, float* dx, float* dgamma, float* dbeta) {
  const int chunks = (d.S + kRows - 1) / kRows;
  vtlb_workspace ws(ctx);
  void* scratch = nullptr;
  const size_t sums = (size_t)d.B * chunks * d.C * sizeof(double2);
  if (int rc = ws.get(sums + (size_t)d.B * d.G * sizeof(float2), &scratch)) return rc;
  double2* partial = (double2*)scratch;
  float2* coef = (float2*)((char*)scratch + sums);
  gn_sums_kernel<ACT, true><<<dim3((d.C + 31) / 32, chunks, d.B), 256, 0, ctx->stream>>>(x, g, gamma, beta, mean, rstd, d,
                                                                                         partial);
  VTLB_LAUNCHED(ctx);
  if (dgamma || dbeta) {
    gn_params_kernel<<<(d.C + 63) / 64, 64, 0, ctx->stream>>>(partial, d.B * chunks, d.C, dgamma, dbeta);
    VTLB_LAUNCHED(ctx);
  }
  if (!dx) return VTLB_OK;
  gn_groups_kernel<true><<<(unsigned)(((size_t)d.B * d.G + 7) / 8), 256, 0, ctx->stream>>>(partial, chunks, d, gamma, 0.0,
                                                                                           nullptr, nullptr, coef);
  VTLB_LAUNCHED(ctx);
  gn_apply_kernel<ACT, true><<<ctx->sm_count * 8, 256, 0, ctx->stream>>>(x, g, gamma, beta, mean, rstd, coef, d, dx);
  VTLB_LAUNCHED(ctx);
  return VTLB_OK;
}

}  // namespace

VTLB_API int vtlb_groupnorm_fwd_f32(vtlb_ctx* ctx, const void* d_x, int B, int S, int C, int groups,
                                    const void* d_gamma_or_null, const void* d_beta_or_null, double eps, int act_kind,
                                    void* d_y, void* d_mean, void* d_rstd) {
  VTLB_ENTER(ctx);
  GnDims d;
  if (int rc = check_dims(ctx, "vtlb_groupnorm_fwd_f32", B, S, C, groups, act_kind, &d)) return rc;
  if (!(eps >= 0.0)) return vtlb_fail(ctx, VTLB_EINVAL, "vtlb_groupnorm_fwd_f32: eps must not be negative");
  if (!d_x || !d_y || !d_mean || !d_rstd) return vtlb_fail(ctx, VTLB_EINVAL, "vtlb_groupnorm_fwd_f32: null pointer");
  const size_t n = (size_t)B * S * C;
  if (d_x != d_y && vtlb_overlap(d_x, n, d_y, n))
    return vtlb_fail(ctx, VTLB_EINVAL, "vtlb_groupnorm_fwd_f32: input and result overlap in part");
  const float *x = (const float*)d_x, *ga = (const float*)d_gamma_or_null, *be = (const float*)d_beta_or_null;
  float *y = (float*)d_y, *mean = (float*)d_mean, *rstd = (float*)d_rstd;
  if (act_kind == VTLB_ACT_RELU) return gn_forward<VTLB_ACT_RELU>(ctx, x, d, ga, be, eps, y, mean, rstd);
  if (act_kind == VTLB_ACT_SILU) return gn_forward<VTLB_ACT_SILU>(ctx, x, d, ga, be, eps, y, mean, rstd);
  return gn_forward<VTLB_ACT_NONE>(ctx, x, d, ga, be, eps, y, mean, rstd);
}

VTLB_API int vtlb_groupnorm_bwd_f32(vtlb_ctx* ctx, const void* d_g, const void* d_x, int B, int S, int C, int groups,
                                    const void* d_gamma_or_null, const void* d_beta_or_null, const void* d_mean,
                                    const void* d_rstd, int act_kind, void* d_dx_or_null, void* d_dgamma_or_null,
                                    void* d_dbeta_or_null) {
  VTLB_ENTER(ctx);
  GnDims d;
  if (int rc = check_dims(ctx, "vtlb_groupnorm_bwd_f32", B, S, C, groups, act_kind, &d)) return rc;
  if (!d_g || !d_x || !d_mean || !d_rstd) return vtlb_fail(ctx, VTLB_EINVAL, "vtlb_groupnorm_bwd_f32: null pointer");
  const size_t n = (size_t)B * S * C;
  if (d_dx_or_null && ((d_dx_or_null != d_x && vtlb_overlap(d_x, n, d_dx_or_null, n)) ||
                       (d_dx_or_null != d_g && vtlb_overlap(d_g, n, d_dx_or_null, n))))
    return vtlb_fail(ctx, VTLB_EINVAL, "vtlb_groupnorm_bwd_f32: an input and dx overlap in part");
  const float *g = (const float*)d_g, *x = (const float*)d_x, *ga = (const float*)d_gamma_or_null;
  const float *be = (const float*)d_beta_or_null, *mean = (const float*)d_mean, *rstd = (const float*)d_rstd;
  float *dx = (float*)d_dx_or_null, *dgamma = (float*)d_dgamma_or_null, *dbeta = (float*)d_dbeta_or_null;
  if (act_kind == VTLB_ACT_RELU)
    return gn_backward<VTLB_ACT_RELU>(ctx, g, x, d, ga, be, mean, rstd, dx, dgamma, dbeta);
  if (act_kind == VTLB_ACT_SILU)
    return gn_backward<VTLB_ACT_SILU>(ctx, g, x, d, ga, be, mean, rstd, dx, dgamma, dbeta);
  return gn_backward<VTLB_ACT_NONE>(ctx, g, x, d, ga, be, mean, rstd, dx, dgamma, dbeta);
}
