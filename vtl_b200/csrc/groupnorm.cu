// Group norm with an activation, channels last: x[B, S, C] (S positions: H * W of a feature map, the length of a
// sequence, 1 for plain features), C channels in `groups` equal groups.  Per sample and group, over S * C/groups values,
//   h = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps) (biased variance),  z = gamma_c * h + beta_c,  y = act(z).
// Backward, with dz = g * act'(z) and n = S * C/groups:
//   dgamma_c = sum over samples and positions of dz * h,   dbeta_c = sum of dz,
//   dx = rstd * (gamma_c * dz - (sum gamma dz) / n - h * (sum gamma dz h) / n), the sums over the group.
#include <cooperative_groups.h>

#include "common.cuh"
#include "gemm_tc.cuh"
#include "groupnorm_plan.h"
#include "ptx.cuh"

namespace {

struct GnDims {
  int B, S, C, G, width;  // width = C / G
};

template <int VEC>
struct GnVec {
  float e[VEC];
};
template <int VEC>
__device__ __forceinline__ GnVec<VEC> gn_load(const float* p) {
  GnVec<VEC> v;
  if constexpr (VEC == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v.e[0] = f.x, v.e[1] = f.y, v.e[2] = f.z, v.e[3] = f.w;
  } else {
    v.e[0] = *p;
  }
  return v;
}
template <int VEC>
__device__ __forceinline__ void gn_store(float* p, const GnVec<VEC>& v) {
  if constexpr (VEC == 4)
    *reinterpret_cast<float4*>(p) = make_float4(v.e[0], v.e[1], v.e[2], v.e[3]);
  else
    *p = v.e[0];
}

// Two f32 operations in one instruction (each rounded as the scalar one is): the kernels below are bound by what the
// schedulers issue before they are bound by HBM.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
template <int VEC>
__device__ __forceinline__ GnVec<VEC> gn_splat(float x) {
  GnVec<VEC> r;
#pragma unroll
  for (int k = 0; k < VEC; ++k) r.e[k] = x;
  return r;
}
#define VTLB_GN_VEC_OP(NAME, PARAMS, PAIR, SINGLE)                                                                        \
  template <int VEC>                                                                                                      \
  __device__ __forceinline__ GnVec<VEC> NAME PARAMS {                                                                     \
    GnVec<VEC> r;                                                                                                         \
    if constexpr (VEC == 4) {                                                                                             \
      _Pragma("unroll") for (int k = 0; k < 4; k += 2) {                                                                  \
        const float2 t = unpack2(PAIR);                                                                                   \
        r.e[k] = t.x, r.e[k + 1] = t.y;                                                                                   \
      }                                                                                                                   \
    } else {                                                                                                              \
      const int k = 0;                                                                                                    \
      r.e[0] = SINGLE;                                                                                                    \
    }                                                                                                                     \
    return r;                                                                                                             \
  }
#define VTLB_GN_PAIR(v) pack2(v.e[k], v.e[k + 1])
VTLB_GN_VEC_OP(vadd, (const GnVec<VEC>& a, const GnVec<VEC>& b), add2(VTLB_GN_PAIR(a), VTLB_GN_PAIR(b)),
               __fadd_rn(a.e[k], b.e[k]))
VTLB_GN_VEC_OP(vmul, (const GnVec<VEC>& a, const GnVec<VEC>& b), mul2(VTLB_GN_PAIR(a), VTLB_GN_PAIR(b)),
               __fmul_rn(a.e[k], b.e[k]))
VTLB_GN_VEC_OP(vfma, (const GnVec<VEC>& a, const GnVec<VEC>& b, const GnVec<VEC>& c),
               fma2(VTLB_GN_PAIR(a), VTLB_GN_PAIR(b), VTLB_GN_PAIR(c)), fmaf(a.e[k], b.e[k], c.e[k]))
#undef VTLB_GN_PAIR
#undef VTLB_GN_VEC_OP
template <int VEC>
__device__ __forceinline__ GnVec<VEC> vneg(const GnVec<VEC>& a) {
  GnVec<VEC> r;
#pragma unroll
  for (int k = 0; k < VEC; ++k) r.e[k] = -a.e[k];
  return r;
}

// e = exp(-z) and s = 1 / (1 + e); expf and IEEE division take some twenty instructions, more than the rest of the forward
// kernel per element.  e is held at 2^127 at most, whose reciprocal, a subnormal, is flushed to zero: for z below -87.3 s
// and e * s are zero, as they are but for 1e-38, whatever multiple of z they are multiplied by.
// In half steps (2^-24, relative): the product z * log2(e) is rounded, which weighs |z| in the power; the approximate
// power is good to 2 ulp, the sum to half an ulp, the approximate reciprocal to 1 ulp: |z| + 4 + 1 + 2 for s, less for
// z > 0.  (A power on the FMA pipe for one element of four and one reciprocal for two were tried: no gain, the kernels
// wait for HBM.)
template <int VEC>
__device__ __forceinline__ void vlogistic(const GnVec<VEC>& z, GnVec<VEC>& e, GnVec<VEC>& s) {
  e = vmul(z, gn_splat<VEC>(-1.4426950408889634f));
#pragma unroll
  for (int k = 0; k < VEC; ++k) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.e[k]) : "f"(fminf(e.e[k], 127.0f)));
  s = vadd(e, gn_splat<VEC>(1.0f));
#pragma unroll
  for (int k = 0; k < VEC; ++k) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.e[k]) : "f"(s.e[k]));
}

template <int ACT, int VEC>
__device__ __forceinline__ GnVec<VEC> act(GnVec<VEC> z) {
  if (ACT == VTLB_ACT_RELU) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) z.e[k] = z.e[k] < 0.0f ? 0.0f : z.e[k];
  }
  if (ACT == VTLB_ACT_SILU) {
    GnVec<VEC> e, s;
    vlogistic(z, e, s);
    return vmul(z, s);
  }
  return z;
}

// g * act'(z), z = gamma * h + beta.  ReLU passes the gradient at exactly zero (nn/internal/activation.v:78-87); z close to
// zero is evaluated again in f64: rounding must not decide which side it is on.
template <int ACT, int VEC>
__device__ __forceinline__ GnVec<VEC> act_bwd(GnVec<VEC> g, const GnVec<VEC>& x, const GnVec<VEC>& mean, const GnVec<VEC>& rstd,
                                              const GnVec<VEC>& gamma, const GnVec<VEC>& beta, const GnVec<VEC>& h) {
  if (ACT == VTLB_ACT_RELU) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const float a = __fmul_rn(gamma.e[k], h.e[k]), z = __fadd_rn(a, beta.e[k]);
      if (fabsf(z) <= 1e-6f * (fabsf(a) + fabsf(beta.e[k]))) {
        const double zd = ((double)x.e[k] - (double)mean.e[k]) * (double)rstd.e[k] * (double)gamma.e[k] + (double)beta.e[k];
        g.e[k] = zd < 0.0 ? 0.0f : g.e[k];
      } else {
        g.e[k] = z < 0.0f ? 0.0f : g.e[k];
      }
    }
    return g;
  }
  if (ACT == VTLB_ACT_SILU) {
    const GnVec<VEC> z = vfma(gamma, h, beta);
    GnVec<VEC> e, s;
    vlogistic(z, e, s);
    return vmul(g, vfma(s, vmul(z, vmul(e, s)), s));  // s + s * z * (1 - s), and 1 - s = e * s without cancellation
  }
  return g;
}

// 1 / sqrt(v), v >= 0, rounded from a value good to 2^-40: an approximate root and one Newton step in f64, a tenth of the
// time of f64 division and root, which every CTA would sit through between two barriers.
__device__ __forceinline__ float inv_sqrt(double v) {
  if (!(v > 1e-30 && v < 1e30)) return (float)(1.0 / sqrt(v));
  const double r = (double)rsqrtf((float)v);
  return (float)(r * fma(-0.5 * v * r, r, 1.5));
}

// ---------------------------------------------------------------- one position per sample
// Plain features and tokens (a layer norm, where there is one group): a group is one row of `width` values next to one
// another.  L threads hold it, PER pieces of VEC each, and a CTA of 256 holds 256 / L rows, so that no thread idles and
// no cluster is kept for a kilobyte.  Bound by HBM, 8 bytes per element forward, 12 backward: 10000 rows of 4096 52 us, 6.4 TB/s, and
// 101 us, 4.9 TB/s (by the clusters below, which pay for an exchange per row, 248 and 531); 500000 of 64 40 and 84 us (2707
// and 4730); 65536 of 32 groups of 32 with SiLU 127 and 216 us.
constexpr int kGnRowThreads = 256;
template <int L>
__device__ __forceinline__ float2 gn_row_sum(float2 v, float2* sm, int turn) {  // over the L threads of a row
#pragma unroll
  for (int o = (L < 32 ? L : 32) / 2; o; o >>= 1) v.x += __shfl_xor_sync(~0u, v.x, o), v.y += __shfl_xor_sync(~0u, v.y, o);
  if constexpr (L > 32) {
    float2* box = sm + turn * (kGnRowThreads / 32);  // (two in turn: the next but one sum is written behind a barrier)
    if ((threadIdx.x & 31) == 0) box[threadIdx.x >> 5] = v;
    __syncthreads();
    box += threadIdx.x / L * (L / 32);
    v = box[0];
#pragma unroll
    for (int q = 1; q < L / 32; ++q) v.x += box[q].x, v.y += box[q].y;
  }
  return v;
}

template <int ACT, int VEC, int L, int PER>
__global__ void __launch_bounds__(kGnRowThreads) gn_rows_fwd_kernel(const float* x, const float* gamma, const float* beta, GnDims d,
                                                                    float eps, double part, float* y, float* mean_out, float* rstd_out) {
  __shared__ float2 sm[2 * kGnRowThreads / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int t = threadIdx.x % L, W = d.width;
  const size_t row = blockIdx.x * (size_t)(kGnRowThreads / L) + threadIdx.x / L;
  const bool in = row < (size_t)d.B * d.G;
  const float* from = x + row * W;
  GnVec<VEC> v[PER];
  GnVec<VEC> s1 = gn_splat<VEC>(0.0f), s2 = s1;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = (i * L + t) * VEC;
    v[i] = in && e < W ? gn_load<VEC>(from + e) : gn_splat<VEC>(0.0f);
    s1 = vadd(s1, v[i]);
  }
  float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int k = 0; k < VEC; ++k) s.x += s1.e[k];
  const float m0 = gn_row_sum<L>(s, sm, 0).x * (float)part;  // the mean but for its rounding; then the distances from it
  const GnVec<VEC> minus0 = gn_splat<VEC>(-m0);
  s1 = gn_splat<VEC>(0.0f);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if ((i * L + t) * VEC >= W) break;
    const GnVec<VEC> a = vadd(v[i], minus0);
    s1 = vadd(s1, a);
    s2 = vfma(a, a, s2);
  }
  s = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int k = 0; k < VEC; ++k) s.x += s1.e[k], s.y += s2.e[k];
  s = gn_row_sum<L>(s, sm, 1);
  // (in f64: of values that hardly vary the distances are exact, and all of them may be what m0 was rounded by)
  const double off = (double)s.x * part, var = fma((double)s.y, part, -off * off);
  const float mu = (float)((double)m0 + off), rs = 1.0f / sqrtf((float)(var < 0.0 ? 0.0 : var) + eps);
  if (!in) return;
  if (t == 0) mean_out[row] = mu, rstd_out[row] = rs;
  const GnVec<VEC> minus = gn_splat<VEC>(-mu), scale = gn_splat<VEC>(rs);
  const int c0 = (int)(row % d.G) * W;
  float* to = y + row * W;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = (i * L + t) * VEC;
    if (e >= W) break;
    const GnVec<VEC> ga = gamma ? gn_load<VEC>(gamma + c0 + e) : gn_splat<VEC>(1.0f);
    const GnVec<VEC> be = beta ? gn_load<VEC>(beta + c0 + e) : gn_splat<VEC>(0.0f);
    gn_store<VEC>(to + e, act<ACT>(vfma(vmul(vadd(v[i], minus), scale), ga, be)));
  }
}

// A CTA takes `each` rows of one group per place for a row, and leaves one row of sums for dgamma and dbeta (at most 64 rows
// are added in f32, the places and, in gn_params_kernel, the CTAs in f64).
template <int ACT, int VEC, int L, int PER>
__global__ void __launch_bounds__(kGnRowThreads, PER > 4 ? 1 : 2)
    gn_rows_bwd_kernel(const float* g, const float* x, const float* gamma, const float* beta, const float* mean, const float* rstd,
                       GnDims d, int each, float* dx, float2* sums) {
  constexpr int R = kGnRowThreads / L;
  __shared__ float2 sm[2 * kGnRowThreads / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int t = threadIdx.x % L, place = threadIdx.x / L, W = d.width;
  const int group = (int)(blockIdx.x % d.G), chunk = (int)(blockIdx.x / d.G), c0 = group * W;
  const float part = 1.0f / (float)W;
  GnVec<VEC> sum1[PER], sum2[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) sum1[i] = sum2[i] = gn_splat<VEC>(0.0f);
  const long long first = (long long)chunk * each * R, end = min((long long)d.B, first + (long long)each * R);
  constexpr bool AHEAD = PER <= 4;  // the next row is fetched while this one is worked on, where the registers allow
  GnVec<VEC> vx[PER], vg[PER], nx[PER], ng[PER];
  float mu_next = 0.0f, rs_next = 0.0f;
  const auto fetch = [&](GnVec<VEC>(&vx)[PER], GnVec<VEC>(&vg)[PER], long long b) {
    const size_t row = (size_t)b * d.G + group;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = (i * L + t) * VEC;
      vx[i] = vg[i] = gn_splat<VEC>(0.0f);
      if (b < end && e < W) vx[i] = gn_load<VEC>(x + row * W + e), vg[i] = gn_load<VEC>(g + row * W + e);
    }
    if (b < end) mu_next = mean[row], rs_next = rstd[row];
  };
  fetch(nx, ng, first + place);
  for (long long b0 = first, k = 0; b0 < end; b0 += R, ++k) {
    const bool in = b0 + place < end;
    const size_t row = (size_t)(b0 + place) * d.G + group;
    const GnVec<VEC> mu = gn_splat<VEC>(mu_next), rs = gn_splat<VEC>(rs_next), minus = vneg(mu);
#pragma unroll
    for (int i = 0; i < PER; ++i) vx[i] = nx[i], vg[i] = ng[i];
    if (AHEAD) fetch(nx, ng, b0 + R + place);
    GnVec<VEC> s1 = gn_splat<VEC>(0.0f), s2 = s1;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = (i * L + t) * VEC;
      if (!in || e >= W) break;
      const GnVec<VEC> ga = gamma ? gn_load<VEC>(gamma + c0 + e) : gn_splat<VEC>(1.0f);
      const GnVec<VEC> be = beta ? gn_load<VEC>(beta + c0 + e) : gn_splat<VEC>(0.0f);
      const GnVec<VEC> h = vmul(vadd(vx[i], minus), rs), dz = act_bwd<ACT>(vg[i], vx[i], mu, rs, ga, be, h);
      sum1[i] = vadd(sum1[i], dz);
      sum2[i] = vfma(dz, h, sum2[i]);
      vx[i] = h;
      vg[i] = vmul(dz, ga);
      s1 = vadd(s1, vg[i]);
      s2 = vfma(vg[i], h, s2);
    }
    if (dx) {
      float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int q = 0; q < VEC; ++q) s.x += s1.e[q], s.y += s2.e[q];
      s = gn_row_sum<L>(s, sm, (int)k & 1);
      const GnVec<VEC> m1 = gn_splat<VEC>(-s.x * part), m2 = gn_splat<VEC>(-s.y * part);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int e = (i * L + t) * VEC;
        if (!in || e >= W) break;
        gn_store<VEC>(dx + row * W + e, vmul(rs, vadd(vg[i], vfma(vx[i], m2, m1))));
      }
    }
    if (!AHEAD) fetch(nx, ng, b0 + R + place);
  }
  if (!sums) return;
  float2* out = sums + (size_t)chunk * d.C + c0;
  if constexpr (R > 1) {
    constexpr int kRow = L * PER * VEC;
    __shared__ float2 box[R * kRow];
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int q = 0; q < VEC; ++q) box[place * kRow + (i * L + t) * VEC + q] = make_float2(sum1[i].e[q], sum2[i].e[q]);
    __syncthreads();
    for (int e = threadIdx.x; e < W; e += kGnRowThreads) {
      double2 s = make_double2(0.0, 0.0);
      for (int q = 0; q < R; ++q) s.x += (double)box[q * kRow + e].x, s.y += (double)box[q * kRow + e].y;
      out[e] = make_float2((float)s.x, (float)s.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = (i * L + t) * VEC;
      if (e >= W) break;
#pragma unroll
      for (int q = 0; q < VEC; ++q) out[e + q] = make_float2(sum1[i].e[q], sum2[i].e[q]);
    }
  }
}

// ---------------------------------------------------------------- groups of any size
// Two passes over x (and g): sums per channel and chunk of positions, then the result.  CTAs take 256 threads as
// `cols` pieces of VEC channels by 256 / cols rows.  Sums are f64: forward of the distances from the group's first value,
// and of their squares (of the values themselves the variance would lose 2^-53 of the mean square, 1e-4 at a mean of 1e6),
// rows that are asked for together by way of the first of them in f32; backward dz and dz * h.
// Bound by HBM, 12 bytes per element forward, 20 backward, less what of x and g still lies in L2 for the second pass.
// Ten samples of 20000 positions by one group of 64 channels: 35 us forward, 55 us backward, 4.4 and 4.7 TB/s of those bytes.
// Sixty of 4000 by two groups of 31 (rows on no 16-byte boundary, one channel a load): 42 and 71 us, 4.2 TB/s.
constexpr int kRows = 256;  // positions per chunk, fewer where there would be too few CTAs

struct GnGrid {
  GnDims d;
  int shift;  // log2 of the pieces per CTA
  int rows;   // positions per chunk
  int across;  // CTAs side by side
};

// Rows that a thread asks for before it uses the first one.  (The result may lie where x or g does, so the compiler would
// not move a load in front of a store: 2.4 TB/s.)
template <int VEC>
constexpr int gn_ahead = VEC == 4 ? 4 : 8;
template <int VEC>
__device__ __forceinline__ void gn_rows(GnVec<VEC> (&v)[gn_ahead<VEC>], const float* from, int r, int r1, int lanes, int C) {
#pragma unroll
  for (int i = 0; i < gn_ahead<VEC>; ++i) {
    if (r + i * lanes < r1) v[i] = gn_load<VEC>(from + (size_t)(r + i * lanes) * C);
  }
}

template <int ACT, bool BWD, int VEC>
__global__ void __launch_bounds__(256) gn_sums_kernel(const float* x, const float* g, const float* gamma,
                                                      const float* beta, const float* mean, const float* rstd, GnGrid t,
                                                      double2* partial) {
  __shared__ double2 sm[256 * VEC];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const GnDims d = t.d;
  const int cols = 1 << t.shift, lanes = 256 >> t.shift, col = threadIdx.x & (cols - 1), lane = threadIdx.x >> t.shift;
  const int b = (int)(blockIdx.x / t.across), c0 = (int)(blockIdx.x % t.across) * cols * VEC, c = c0 + col * VEC, chunk = blockIdx.y;
  const int r1 = min(d.S, (chunk + 1) * t.rows);
  double2 acc[VEC] = {};
  if (c < d.C) {
    GnVec<VEC> mu = {}, rs = {}, ga = {}, be = {};
    if (BWD) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const size_t st = (size_t)b * d.G + (c + k) / d.width;
        mu.e[k] = mean[st], rs.e[k] = rstd[st];
        ga.e[k] = gamma ? gamma[c + k] : 1.0f, be.e[k] = beta ? beta[c + k] : 0.0f;
      }
    }
    const GnVec<VEC> minus = vneg(mu);
    const size_t base = (size_t)b * d.S * d.C + c;
    double first[VEC] = {};
    for (int r = chunk * t.rows + lane, start = r; r < r1; r += gn_ahead<VEC> * lanes) {
      GnVec<VEC> vx[gn_ahead<VEC>], vg[gn_ahead<VEC>];
      gn_rows<VEC>(vx, x + base, r, r1, lanes, d.C);
      if (BWD) {
        gn_rows<VEC>(vg, g + base, r, r1, lanes, d.C);
#pragma unroll
        for (int i = 0; i < gn_ahead<VEC>; ++i) {
          if (r + i * lanes >= r1) break;
          const GnVec<VEC> h = vmul(vadd(vx[i], minus), rs);
          const GnVec<VEC> dz = act_bwd<ACT>(vg[i], vx[i], mu, rs, ga, be, h);
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            acc[k].x += (double)dz.e[k];
            acc[k].y = fma((double)dz.e[k], (double)h.e[k], acc[k].y);
          }
        }
      } else {
        if (r == start) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) first[k] = (double)x[(size_t)b * d.S * d.C + (d.G == 1 ? 0 : (c + k) / d.width * d.width)];
        }
        if (r + lanes >= r1) {  // one row
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            const double off = (double)vx[0].e[k] - first[k];
            acc[k].x += off, acc[k].y = fma(off, off, acc[k].y);
          }
          break;
        }
        // Distances from the first of these rows, `off` from the group's.  (Where that row is far from the others, its
        // own distance from the mean counts for more than what theirs from it are rounded by.)
        const GnVec<VEC> from = vneg(vx[0]);
        GnVec<VEC> s1 = gn_splat<VEC>(0.0f), s2 = s1;
        float n = 1.0f;
#pragma unroll
        for (int i = 1; i < gn_ahead<VEC>; ++i) {
          if (r + i * lanes >= r1) break;
          const GnVec<VEC> e = vadd(vx[i], from);
          s1 = vadd(s1, e);
          s2 = vfma(e, e, s2);
          n += 1.0f;
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const double off = (double)vx[0].e[k] - first[k], all = (double)n * off, rest = (double)s1.e[k];
          acc[k].x += all + rest;
          acc[k].y += fma(all + (rest + rest), off, (double)s2.e[k]);
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) sm[threadIdx.x * VEC + k] = acc[k];
  __syncthreads();
  for (int i = threadIdx.x; i < cols * VEC; i += 256) {
    const int ch = c0 + i;
    if (ch >= d.C) break;
    double2 s = sm[i];
    for (int l = 1; l < lanes; ++l) s.x += sm[l * cols * VEC + i].x, s.y += sm[l * cols * VEC + i].y;
    partial[((size_t)b * gridDim.y + chunk) * d.C + ch] = s;
  }
}

// One CTA per (sample, group), T threads: the sums over chunks and channels, in a fixed order.  (With a warp for each, which
// also divided to find its channels, 79 chunks of 64 channels took 40 us, longer than both passes over x.)
template <bool BWD>
__global__ void __launch_bounds__(256) gn_groups_kernel(const double2* partial, int chunks, GnDims d, const float* x,
                                                        const float* gamma, double eps, float* mean, float* rstd, float2* coef) {
  __shared__ double2 sm[8];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const unsigned k = blockIdx.x, T = blockDim.x;
  const int b = (int)(k / d.G), grp = (int)(k % d.G);
  const int down = T / d.width, along = T % d.width;  // from one entry of a thread to its next
  int row = threadIdx.x / d.width, col = threadIdx.x % d.width;
  double s0 = 0.0, s1 = 0.0;
  const float first = BWD ? 0.0f : x[(size_t)b * d.S * d.C + grp * d.width];
  while (row < chunks) {
    double2 p[8];
    double w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = grp * d.width + col;
      p[i] = row < chunks ? partial[((size_t)b * chunks + row) * d.C + c] : make_double2(0.0, 0.0);
      w[i] = row >= chunks ? 0.0 : BWD && gamma ? (double)gamma[c] : 1.0;
      row += down, col += along;
      if (col >= d.width) col -= d.width, ++row;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s0 = fma(w[i], p[i].x, s0), s1 = fma(w[i], p[i].y, s1);
  }
  for (int o = 16; o; o >>= 1) s0 += __shfl_xor_sync(~0u, s0, o), s1 += __shfl_xor_sync(~0u, s1, o);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = make_double2(s0, s1);
  __syncthreads();
  if (threadIdx.x) return;
  for (unsigned q = 1; q < T / 32; ++q) s0 += sm[q].x, s1 += sm[q].y;
  const double n = (double)d.S * d.width;
  if (BWD) {
    coef[k] = make_float2((float)(s0 / n), (float)(s1 / n));
  } else {
    const double off = s0 / n, var = s1 / n - off * off;
    mean[k] = (float)((double)first + off);
    rstd[k] = (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + eps));
  }
}

// dgamma and dbeta from the channel sums (dz, dz * h): 8 channels and 32 stretches of rows per CTA, so that few loads of a thread
// wait for one another (a few hundred rows as a rule: latency, not bytes: 960 rows of 62 channels 11 us).
template <typename PAIR>
__global__ void __launch_bounds__(256) gn_params_kernel(const PAIR* sums, int rows, int C, float* dgamma, float* dbeta) {
  __shared__ double2 sm[8][8];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int cl = threadIdx.x & 7, c = blockIdx.x * 8 + cl, warp = threadIdx.x >> 5;
  double2 s = make_double2(0.0, 0.0);
  if (c < C) {
#pragma unroll 8
    for (int r = threadIdx.x >> 3; r < rows; r += 32) {
      const PAIR e = sums[(size_t)r * C + c];
      s.x += (double)e.x, s.y += (double)e.y;
    }
  }
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) s.x += __shfl_xor_sync(~0u, s.x, o), s.y += __shfl_xor_sync(~0u, s.y, o);
  if ((threadIdx.x & 31) < 8) sm[warp][cl] = s;
  __syncthreads();
  if (threadIdx.x >= 8 || c >= C) return;
  for (int q = 1; q < 8; ++q) s.x += sm[q][cl].x, s.y += sm[q][cl].y;
  if (dbeta) dbeta[c] = (float)s.x;
  if (dgamma) dgamma[c] = (float)s.y;
}

template <int ACT, bool BWD, int VEC>
__global__ void __launch_bounds__(256) gn_apply_kernel(const float* x, const float* g, const float* gamma,
                                                       const float* beta, const float* mean, const float* rstd,
                                                       const float2* coef, GnGrid t, float* out) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const GnDims d = t.d;
  const int cols = 1 << t.shift, lanes = 256 >> t.shift, col = threadIdx.x & (cols - 1), lane = threadIdx.x >> t.shift;
  const int b = (int)(blockIdx.x / t.across), c0 = (int)(blockIdx.x % t.across) * cols * VEC, c = c0 + col * VEC, chunk = blockIdx.y;
  const int r1 = min(d.S, (chunk + 1) * t.rows);
  if (c >= d.C) return;
  GnVec<VEC> mu, rs, ga, be, c1 = {}, c2 = {};
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const size_t st = (size_t)b * d.G + (c + k) / d.width;
    mu.e[k] = mean[st], rs.e[k] = rstd[st];
    ga.e[k] = gamma ? gamma[c + k] : 1.0f, be.e[k] = beta ? beta[c + k] : 0.0f;
    if (BWD) c1.e[k] = -rs.e[k] * coef[st].x, c2.e[k] = -rs.e[k] * coef[st].y;
  }
  const GnVec<VEC> minus = vneg(mu), a = vmul(ga, rs);
  const size_t base = (size_t)b * d.S * d.C + c;
  for (int r = chunk * t.rows + lane; r < r1; r += gn_ahead<VEC> * lanes) {
    GnVec<VEC> vx[gn_ahead<VEC>], vg[gn_ahead<VEC>];
    gn_rows<VEC>(vx, x + base, r, r1, lanes, d.C);
    if (BWD) gn_rows<VEC>(vg, g + base, r, r1, lanes, d.C);
#pragma unroll
    for (int i = 0; i < gn_ahead<VEC>; ++i) {
      if (r + i * lanes >= r1) break;
      const GnVec<VEC> dist = vadd(vx[i], minus);
      float* to = out + base + (size_t)(r + i * lanes) * d.C;
      if (BWD) {
        const GnVec<VEC> h = vmul(dist, rs);
        gn_store<VEC>(to, vfma(a, act_bwd<ACT>(vg[i], vx[i], mu, rs, ga, be, h), vfma(h, c2, c1)));
      } else {
        gn_store<VEC>(to, act<ACT>(vfma(dist, a, be)));
      }
    }
  }
}

// ---------------------------------------------------------------- groups that fit the registers of a cluster
// x is read once: it stays in registers between the sums and the result (groupnorm_plan.h).  A cluster goes through
// several units (a slab of groups of one sample), the next one's values on their way into shared memory while this
// one's are worked on.  Bound by HBM, 8 bytes per element forward, 12 backward: with SiLU, 32 samples of 64 x 64 positions by
// 512 channels forward in 95 to 97 us, 5.6 TB/s, 86 % of a plain copy's rate (the same loads and stores without the sums: 6.2
// TB/s); 64 of 32 x 32 backward in 74 to 77 us, 5.3 TB/s (the barriers around the sums of a unit are not hidden with two
// CTAs of 256 threads, all that their registers leave room for).  Forward 512 threads with sixteen pieces each: the
// registers of a cluster of four hold 64 x 64 positions of 32 channels, 128 bytes of a row at a time.  Small maps are bound by
// the host: two samples of 8 x 8 by 128 channels 6.5 us forward.  Channels that are no multiple of four come by 4-byte
// cp.async: three samples of 17 x 19 by 330 channels backward in 8.4 to 9 us with both launches, latency throughout.
// Groups whose width is no multiple of four keep sums per channel: 2.9 to 3.9 TB/s.
struct GnTile {
  GnDims d;
  int groups, slabs, csplit, channels, rows;
  unsigned units;  // B * slabs
  uint32_t zero;   // 0, unknown to the compiler (gn_after)
  int boxes, box_rows;  // of a CTA's piece as the tensor map cuts it
  bool in_place;        // y lies over x
};

// How a CTA's piece of a slab lies on its threads.  The same for all slabs but a narrower last one, so the divisions
// are done once per kernel, not once per unit (where they took a third of all instructions).
struct GnShape {
  int groups;         // of the slab
  int in_slab;        // first channel of this CTA, from the slab's first
  int channels;       // of this CTA
  int cols, lanes;    // pieces of VEC channels in a row, rounded up to a power of two; rows per step
  int real;           // pieces that there are: the threads of the others have no rows
  int col, lane;      // this thread's
  int rows;           // of this thread: lane, lane + lanes, ... of the CTA's
  int group;          // of the thread's first channel, within the slab
  bool any;           // whether the CTA has rows at all
  int r0;             // the CTA's first
  size_t inside;      // the thread's first element, from the unit's (first position, first channel of the slab)
  bool even;          // a warp holds whole rows
};
template <int T, int VEC>
__device__ __forceinline__ GnShape gn_shape(const GnTile& t, int groups, int rank) {
  GnShape p;
  p.groups = groups;
  p.in_slab = (rank % t.csplit) * t.channels;
  p.channels = min(t.channels, groups * t.d.width - p.in_slab);
  p.real = p.channels / VEC;
  const int shift = p.real > 1 ? 32 - __clz(p.real - 1) : 0;
  p.cols = 1 << shift;
  p.lanes = T >> shift;
  p.col = threadIdx.x & (p.cols - 1);
  p.lane = threadIdx.x >> shift;
  const int r0 = min(t.d.S, (rank / t.csplit) * t.rows), r1 = min(t.d.S, r0 + t.rows);
  p.any = r0 < r1;
  p.r0 = r0;
  p.rows = p.col < p.real ? max(0, (r1 - r0 - p.lane + p.lanes - 1) >> (31 - __clz(p.lanes))) : 0;
  p.group = (p.in_slab + p.col * VEC) / t.d.width;
  p.inside = (size_t)(r0 + p.lane) * t.d.C + p.in_slab + p.col * VEC;
  p.even = p.cols <= 32;
  return p;
}

// A unit, and the way to the one that this cluster takes next.
struct GnUnit {
  unsigned unit, b, slab;
};
__device__ __forceinline__ GnUnit gn_first(const GnTile& t, unsigned unit) {
  return GnUnit{unit, unit / t.slabs, unit % t.slabs};
}
__device__ __forceinline__ GnUnit gn_next(const GnTile& t, GnUnit u, const GnUnit& stride) {
  u.unit += stride.unit, u.b += stride.b, u.slab += stride.slab;
  if (u.slab >= (unsigned)t.slabs) u.slab -= t.slabs, u.b += 1;
  return u;
}
__device__ __forceinline__ int gn_groups(const GnTile& t, const GnUnit& u) {
  return min(t.groups, t.d.G - (int)u.slab * t.groups);
}
__device__ __forceinline__ size_t gn_base(const GnTile& t, const GnUnit& u) {
  return (size_t)u.b * t.d.S * t.d.C + (size_t)u.slab * t.groups * t.d.width;
}

// The CTAs of a cluster send one another their sums: st.async into a box of the receiver, counted by an mbarrier there.
// (A cluster barrier instead orders every earlier global store as well: each unit then waited for the results of the
// unit before to reach L2.)  Two boxes in turn: a CTA sends for unit n + 2 only once it has everyone's sums of unit
// n + 1, which they send after they have read those of unit n.
template <typename T>
struct GnMail {
  T box[2][kGnMaxCluster][kGnMaxGroups];
  uint64_t full[2];
  uint64_t data;  // the slots are filled (TMA)
  uint32_t abort;
};
__device__ __forceinline__ uint32_t gn_remote(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void gn_post(uint32_t to, uint32_t bar, double2 v) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];" ::"r"(to),
               "l"(__double_as_longlong(v.x)), "l"(__double_as_longlong(v.y)), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void gn_post(uint32_t to, uint32_t bar, float2 v) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(to),
               "r"(__float_as_uint(v.x)), "r"(__float_as_uint(v.y)), "r"(bar)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void gn_mail_init(GnMail<T>& m) {
  if (threadIdx.x == 0) {
    ptx::mbar_init(ptx::smem_u32(&m.full[0]), 1);
    ptx::mbar_init(ptx::smem_u32(&m.full[1]), 1);
    ptx::mbar_init(ptx::smem_u32(&m.data), 1);
    m.abort = 0;
    ptx::fence_barrier_init();
  }
}
// One thread's sum of group g goes to every CTA of the cluster.
template <typename T>
__device__ __forceinline__ void gn_send(GnMail<T>& m, int turn, int rank, int ctas, int g, T v) {
  if (ctas == 1) {
    m.box[turn][0][g] = v;
    return;
  }
  const uint32_t to = ptx::smem_u32(&m.box[turn][rank][g]), bar = ptx::smem_u32(&m.full[turn]);
  for (int r = 0; r < ctas; ++r) gn_post(gn_remote(to, r), gn_remote(bar, r), v);
}
// The first warp waits for the sums of all CTAs (at most two seconds: then the status word says so at the kernel's
// end, and the results are not valid).  `round` counts the units of this CTA.
template <typename T>
__device__ __forceinline__ void gn_receive(GnMail<T>& m, int turn, unsigned round, int ctas, int groups) {
  const uint32_t bar = ptx::smem_u32(&m.full[turn]);
  if (threadIdx.x == 0) ptx::mbar_arrive_expect_tx(bar, (uint32_t)(ctas * groups * sizeof(T)));
  __syncwarp();
  ptx::mbar_wait_bounded(bar, (round >> 1) & 1, &m.abort, 2000000000ull);
  __syncwarp();  // lanes leave the wait one by one
}

// Waits, for at most two seconds, until the slots are filled for unit number `round` of this CTA.
template <typename T>
__device__ __forceinline__ void gn_wait_data(GnMail<T>& m, unsigned round) {
  ptx::mbar_wait_bounded(ptx::smem_u32(&m.data), round & 1, &m.abort, 2000000000ull);
  __syncwarp();  // lanes leave the wait one by one, and a warp that is not whole counts as a whole one at a barrier
}

// Every copy has been waited for, unless a wait ran out: then the one under way gets another second before the CTA and its
// shared memory go.
template <typename T>
__device__ __forceinline__ void gn_last_copies(GnMail<T>& m) {
  if (!*(volatile uint32_t*)&m.abort || threadIdx.x) return;
  for (uint32_t parity = 0; parity < 2; ++parity) {
    uint32_t none = 0;
    ptx::mbar_wait_bounded(ptx::smem_u32(&m.data), parity, &none, 1000000000ull);
  }
}

// Each thread has slots of its own in shared memory, [i][thread], and reads back what it fetched itself.  A slot is
// filled again as soon as it has been read: `after`, a zero made from the values read, is part of the address, so that
// the copy cannot start before they are in registers.
template <int VEC, int VPT>
__device__ __forceinline__ uint32_t gn_after(const GnTile& t, const GnVec<VEC> (&v)[VPT]) {
  uint32_t all = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int k = 0; k < VEC; ++k) all |= __float_as_uint(v[i].e[k]);
  return all & t.zero;
}
template <int T, int VEC, int VPT>
__device__ __forceinline__ void gn_fetch(float* slots, const float* src, const GnTile& t, const GnUnit& u, const GnShape& p,
                                         uint32_t after = 0) {
  const float* from = src + gn_base(t, u) + p.inside;
  const size_t step = (size_t)p.lanes * t.d.C;
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(slots + threadIdx.x * VEC) + after;
#pragma unroll
  for (int i = 0; i < VPT; ++i, from += step)
    if (i < p.rows) {
      if constexpr (VEC == 4)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * T * 16), "l"(from) : "memory");
      else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + i * T * 4), "l"(from) : "memory");
    }
}
// The same piece by TMA: one thread asks for it, and the threads are spared the requests (16 per thread and unit, a fifth
// of the backward kernel's time).  Rows lie t.channels apart; rows behind S and channels behind C arrive as zeros.
__device__ __forceinline__ void gn_fetch_box(float* slots, const CUtensorMap* map, const GnTile& t, const GnUnit& u,
                                             const GnShape& p, uint32_t bar) {
  const int c = (int)u.slab * t.groups * t.d.width + p.in_slab;
  for (int i = 0; i < t.boxes; ++i)
    ptx::tma_load_3d(ptx::smem_u32(slots + (size_t)i * t.box_rows * t.channels), map, c, p.r0 + i * t.box_rows, (int)u.b, bar);
}
template <int VEC, int VPT>
__device__ __forceinline__ void gn_take_box(GnVec<VEC> (&v)[VPT], const float* slots, const GnTile& t, const GnShape& p) {
  const float* from = slots + p.lane * t.channels + p.col * VEC;
  const int step = p.lanes * t.channels;
#pragma unroll
  for (int i = 0; i < VPT; ++i, from += step) {
    if (i < p.rows) {
      v[i] = gn_load<VEC>(from);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[i].e[k] = 0.0f;
    }
  }
}
// Every thread has read its slots, and the copy engine may write them.  The proxy fence is what holds the copies back: a
// barrier alone orders the reads' issue, and a read can wait in a busy shared memory for longer than a copy takes.
__device__ __forceinline__ void gn_slots_read() {
  ptx::fence_proxy_async();
  __syncthreads();
}

template <int T, int VEC, int VPT>
__device__ __forceinline__ void gn_take(GnVec<VEC> (&v)[VPT], const float* slots, int rows) {
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i < rows) {
      v[i] = gn_load<VEC>(slots + (i * T + threadIdx.x) * VEC);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[i].e[k] = 0.0f;
    }
  }
}

// The groups of units that are marked by a negative rstd once more, each by one CTA, behind the barrier of the cluster: sums
// in f64 of the distances from the mean that was found, so that a constant group's variance is zero but for 2^-53 of the
// square of what that mean is rounded by.  x is still there: where y lies over it, marked units were not written.  It takes
// no registers from the way that units take as a rule, which pays for the check at the kernel's end.  x is read twice more, four
// pieces a thread at a time: 32 samples of 64 x 64 x 512 that are all marked 520 us (95 where none is; one piece at a time 1850).
template <int ACT, int T, int V>
__device__ __forceinline__ void gn_look_again(const float* x, const float* gamma, const float* beta, const GnTile& t, int rank, int ctas,
                                           double eps, float* y, float* mean_out, float* rstd_out, double2* sm) {
  __syncthreads();
  const int tid = threadIdx.x, W = t.d.width;
  constexpr int U = 4;
  const int cols = W / V, n = t.d.S * cols;  // pieces (at most what a cluster holds)
  const GnUnit stride = gn_first(t, gridDim.x / ctas);
  for (GnUnit u = gn_first(t, blockIdx.x / ctas); u.unit < t.units; u = gn_next(t, u, stride)) {
    for (int g = rank; g < gn_groups(t, u); g += ctas) {
      const size_t k = (size_t)u.b * t.d.G + u.slab * t.groups + g;
      if (!(*(volatile float*)&rstd_out[k] < 0.0f)) continue;  // (the same for all threads: one writes it, behind a barrier)
      const size_t base = gn_base(t, u) + (size_t)g * W;
      const double near = (double)*(volatile float*)&mean_out[k];
      double2 s = make_double2(0.0, 0.0);
      const auto fetch = [&](GnVec<V>(&v)[U], int e0) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int e = e0 + i * T;
          if (e < n) v[i] = gn_load<V>(x + base + (size_t)(e / cols) * t.d.C + e % cols * V);
        }
      };
#pragma unroll 1
      for (int e = tid; e < n; e += U * T) {
        GnVec<V> v[U];
        fetch(v, e);
#pragma unroll
        for (int i = 0; i < U; ++i) {
          if (e + i * T >= n) break;
#pragma unroll
          for (int q = 0; q < V; ++q) {
            const double far = (double)v[i].e[q] - near;
            s.x += far, s.y = fma(far, far, s.y);
          }
        }
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) s.x += __shfl_xor_sync(~0u, s.x, o), s.y += __shfl_xor_sync(~0u, s.y, o);
      if ((tid & 31) == 0) sm[tid >> 5] = s;
      __syncthreads();
      s = sm[0];
#pragma unroll 1
      for (int q = 1; q < T / 32; ++q) s.x += sm[q].x, s.y += sm[q].y;
      const double all = (double)n * V, off = s.x / all, var = s.y / all - off * off;
      const float mu = (float)(near + off), rs = inv_sqrt((var < 0.0 ? 0.0 : var) + eps);
      if (tid == 0) mean_out[k] = mu, rstd_out[k] = rs;
      const int c0 = ((int)u.slab * t.groups + g) * W;
#pragma unroll 1
      for (int e0 = tid; e0 < n; e0 += U * T) {
        GnVec<V> v[U];
        fetch(v, e0);
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int e = e0 + i * T, c = e % cols * V;
          if (e >= n) break;
#pragma unroll
          for (int q = 0; q < V; ++q)
            v[i].e[q] = fmaf(v[i].e[q] - mu, gamma ? rs * __ldg(gamma + c0 + c + q) : rs, beta ? __ldg(beta + c0 + c + q) : 0.0f);
          gn_store<V>(y + base + (size_t)(e / cols) * t.d.C + c, act<ACT>(v[i]));
        }
      }
      __syncthreads();
    }
  }
}

template <int ACT, int VEC, int VPT, bool GROUPED, bool TMA>
__global__ void __launch_bounds__(kGnFwdThreads, VPT > 8 ? 512 / kGnFwdThreads : 1024 / kGnFwdThreads)
    gn_fwd_tile_kernel(const __grid_constant__ CUtensorMap map, const float* x, const float* gamma, const float* beta, GnTile t, double eps, float* y,
                       float* mean_out, float* rstd_out, uint32_t* status) {
  namespace cg = cooperative_groups;
  constexpr int T = kGnFwdThreads;
  constexpr int PAIRS = GROUPED ? 1 : VEC;  // GROUPED: the channels of a thread's piece are all of one group
  constexpr int PER = VEC / PAIRS;          // channels per pair of sums
  __shared__ double2 sm_pair[T * PAIRS];      // [row lane or warp][entry or group]
  __shared__ GnMail<double2> mail;
  __shared__ float2 sm_stat[kGnMaxGroups];
  __shared__ unsigned sm_lost;  // the last round in which the sums of a group lost too much
  extern __shared__ __align__(128) float slots[];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const int tid = threadIdx.x, warp = tid >> 5, width = t.d.width;
  const GnUnit stride = gn_first(t, gridDim.x / ctas);
  GnUnit u = gn_first(t, blockIdx.x / ctas);
  GnShape p = gn_shape<T, VEC>(t, gn_groups(t, u), rank);
  const int cq = width / PER;  // pairs per group and row
  const bool cq_even = PAIRS == 1 && (cq & (cq - 1)) == 0;
  const double part = 1.0 / ((double)t.d.S * width);
  gn_mail_init(mail);
  if (tid == 0) sm_lost = ~0u;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early: the kernel in front is done from here on
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t bar = ptx::smem_u32(&mail.data), box_bytes = (uint32_t)(t.boxes * t.box_rows * t.channels * 4);
  if constexpr (TMA) {
    if (tid == 0 && p.any) {
      ptx::mbar_arrive_expect_tx(bar, box_bytes);
      gn_fetch_box(slots, &map, t, u, p, bar);
    }
  } else {
    gn_fetch<T, VEC, VPT>(slots, x, t, u, p);
  }
  if (TMA && ctas == 1) __syncthreads();  // (the barrier is ready)
  if (ctas > 1) cluster.sync();  // everyone's boxes are ready
  for (unsigned round = 0;; ++round) {
    const int turn = round & 1;
    GnVec<VEC> v[VPT];
    const GnUnit next = gn_next(t, u, stride);
    if constexpr (TMA) {
      if (p.any) gn_wait_data(mail, round);
      gn_take_box(v, slots, t, p);
      gn_slots_read();
      if (tid == 0 && p.any && next.unit < t.units && !mail.abort) {
        ptx::mbar_arrive_expect_tx(bar, box_bytes);
        gn_fetch_box(slots, &map, t, next, p, bar);  // (in_slab and r0 are those of every slab)
      }
    } else {
      asm volatile("cp.async.wait_all;" ::: "memory");
      gn_take<T>(v, slots, p.rows);
      if (next.unit < t.units) {
        const uint32_t after = gn_after(t, v);
        if (gn_groups(t, next) == p.groups)
          gn_fetch<T, VEC, VPT>(slots, x, t, next, p, after);
        else
          gn_fetch<T, VEC, VPT>(slots, x, t, next, gn_shape<T, VEC>(t, gn_groups(t, next), rank), after);
      }
    }
    // A thread's own mean m, and the sums r and q of the distances from it and of their squares, in f32 (m is rounded, r
    // says by how much); from these in f64 the sums of x and x^2.  Of these the variance loses some 2^-53 of the mean
    // square: where that may be more than 2^-27 of variance and eps (a constant group of 30 at an eps of 1e-5), the unit is
    // left to gn_look_again.  (Sums of the distances from a value that all threads know lose nothing, but it has to
    // be brought and subtracted for every unit: 26 samples of 129 x 896 by 16 groups 12.0 us, this way 11.6 to 11.9, sums
    // without care 11.0; 32 of 64 x 64 x 512 96, 95 and 93.)
    double2 acc[PAIRS];
    {
      const float n = (float)(p.rows * PER), part_n = p.rows ? __fdividef(1.0f, n) : 0.0f;
      GnVec<VEC> m = gn_splat<VEC>(0.0f), r = m, q = m;
#pragma unroll
      for (int i = 0; i < VPT; ++i) m = vadd(m, v[i]);
      if constexpr (PAIRS == 1) {
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum += m.e[k];
        m = gn_splat<VEC>(sum * part_n);  // any value near the mean serves
      } else {
        m = vmul(m, gn_splat<VEC>(part_n));
      }
      const GnVec<VEC> minus = vneg(m);
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (i < p.rows) {
          const GnVec<VEC> e = vadd(v[i], minus);
          r = vadd(r, e);
          q = vfma(e, e, q);
        }
#pragma unroll
      for (int k = 0; k < PAIRS; ++k) {
        if constexpr (PAIRS == 1) {
#pragma unroll
          for (int e = 1; e < VEC; ++e) r.e[0] += r.e[e], q.e[0] += q.e[e];
        }
        const double rest = (double)r.e[k], s = fma((double)n, (double)m.e[k], rest);
        acc[k] = make_double2(s, fma(s + rest, (double)m.e[k], (double)q.e[k]));
      }
    }
    // The pairs of all rows, per entry (a piece, or a channel of it): by shuffles where a warp holds whole rows.
    const int entries = p.cols * PAIRS, parts = p.even ? T / 32 : p.lanes;  // of a row; rows of sums
    const bool whole = p.even && cq_even && cq <= p.cols;  // a group is some lanes of a warp: its entries by shuffles too
    if (p.even) {
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        if (o >= p.cols || (whole && o < cq)) {
#pragma unroll
          for (int q = 0; q < PAIRS; ++q) {
            acc[q].x += __shfl_xor_sync(~0u, acc[q].x, o);
            acc[q].y += __shfl_xor_sync(~0u, acc[q].y, o);
          }
        }
      }
      const int lane = tid & 31;
      if (whole) {
        if (lane < p.real && (lane & (cq - 1)) == 0) sm_pair[warp * p.groups + p.group] = acc[0];
      } else if (lane < p.cols) {
#pragma unroll
        for (int q = 0; q < PAIRS; ++q) sm_pair[warp * entries + lane * PAIRS + q] = acc[q];
      }
    } else {
#pragma unroll
      for (int q = 0; q < PAIRS; ++q) sm_pair[tid * PAIRS + q] = acc[q];
    }
    __syncthreads();
    if (whole) {
      if (tid < p.groups) {
        double2 s = sm_pair[tid];
#pragma unroll
        for (int w = 1; w < T / 32; ++w) s.x += sm_pair[w * p.groups + tid].x, s.y += sm_pair[w * p.groups + tid].y;
        gn_send(mail, turn, rank, ctas, tid, s);
      }
    } else {
      // A thread per entry adds up the rows of sums; then one warp per group of the slab, its entries in this CTA.
      for (int e = tid; parts > 1 && e < entries; e += T) {
        double2 s = sm_pair[e];
#pragma unroll 5
        for (int q = 1; q < parts; ++q) s.x += sm_pair[q * entries + e].x, s.y += sm_pair[q * entries + e].y;
        sm_pair[e] = s;
      }
      if (parts > 1) __syncthreads();
      for (int g = warp; g < p.groups; g += T / 32) {
        const int lo = max(g * width - p.in_slab, 0) / PER, hi = min((g + 1) * width - p.in_slab, p.channels) / PER;
        double2 s = make_double2(0.0, 0.0);
        for (int e = lo + (tid & 31); e < hi; e += 32) s.x += sm_pair[e].x, s.y += sm_pair[e].y;
#pragma unroll
        for (int o = 16; o; o >>= 1) s.x += __shfl_xor_sync(~0u, s.x, o), s.y += __shfl_xor_sync(~0u, s.y, o);
        if ((tid & 31) == 0) gn_send(mail, turn, rank, ctas, g, s);
      }
      if (ctas == 1) __syncthreads();
    }
    if (warp == 0 && ctas > 1) gn_receive(mail, turn, round, ctas, p.groups);
    if (tid < p.groups) {
      double2 s = make_double2(0.0, 0.0);
      for (int r = 0; r < ctas; ++r) s.x += mail.box[turn][r][tid].x, s.y += mail.box[turn][r][tid].y;
      const double off = s.x * part, var = s.y * part - off * off;
      const float2 st = make_float2((float)off, inv_sqrt((var < 0.0 ? 0.0 : var) + eps));
      sm_stat[tid] = st;
      const bool lost = __any_sync(~0u >> (32 - p.groups), fabsf(st.x) * st.y > 8192.0f);
      if (lost) sm_lost = round;
      if (rank == 0) {
        const size_t k = (size_t)u.b * t.d.G + u.slab * t.groups + tid;
        mean_out[k] = st.x;
        rstd_out[k] = lost ? -st.y : st.y;  // (a mark for gn_look_again)
      }
    }
    __syncthreads();
    if (p.rows && !(t.in_place && sm_lost == round)) {
      const int c = (int)u.slab * t.groups * width + p.in_slab + p.col * VEC;
      GnVec<VEC> minus, a, be;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float2 st = sm_stat[GROUPED ? p.group : (p.in_slab + p.col * VEC + k) / width];
        minus.e[k] = -st.x;
        a.e[k] = gamma ? st.y * __ldg(gamma + c + k) : st.y;
        be.e[k] = beta ? __ldg(beta + c + k) : 0.0f;
      }
      float* to = y + gn_base(t, u) + p.inside;
      const size_t step = (size_t)p.lanes * t.d.C;
#pragma unroll
      for (int i = 0; i < VPT; ++i, to += step) {
        if (i >= p.rows) break;
        gn_store<VEC>(to, act<ACT>(vfma(vadd(v[i], minus), a, be)));
      }
    }
    if (next.unit >= t.units) break;
    u = next;
    if (gn_groups(t, u) != p.groups) p = gn_shape<T, VEC>(t, gn_groups(t, u), rank);
  }
  if (TMA || ctas > 1) ptx::report_abort(&mail.abort, status, VTLB_ST_NORM_TIMEOUT);  // whichever thread's wait it was
  if (TMA && p.any) gn_last_copies(mail);
  if (ctas > 1) cluster.sync();  // no CTA leaves while another may still send to it
  if (__builtin_expect(sm_lost != ~0u, 0)) gn_look_again<ACT, T, GROUPED ? VEC : 1>(x, gamma, beta, t, (int)cluster.block_rank(), (int)cluster.num_blocks(), eps, y, mean_out, rstd_out, sm_pair);
}

// Backward.  The channel sums of each CTA go to `sums` [B * rsplit][C] (dz, dz * h) for gn_params_kernel.
template <int ACT, int VEC, int VPT, bool GROUPED, bool TMA>
__global__ void __launch_bounds__(kGnBwdThreads, VPT > 4 ? 512 / kGnBwdThreads : 1024 / kGnBwdThreads)
    gn_bwd_tile_kernel(const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_x, const float* g, const float* x, const float* gamma, const float* beta, const float* mean,
                       const float* rstd, GnTile t, float* dx, float2* sums, uint32_t* status) {
  namespace cg = cooperative_groups;
  constexpr int T = kGnBwdThreads;
  __shared__ float2 sm_part[T * VEC];  // [channel], weighted
  __shared__ float2 sm_chan[T * VEC];  // [row lane or warp][channel]
  __shared__ GnMail<float2> mail;
  __shared__ float2 sm_coef[kGnMaxGroups];
  extern __shared__ __align__(128) float slots[];
  const uint32_t bar = ptx::smem_u32(&mail.data), box_bytes = (uint32_t)(t.boxes * t.box_rows * t.channels * 4);
  float* slots_g = slots + (TMA ? box_bytes / 4 : VPT * T * VEC);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const int tid = threadIdx.x, warp = tid >> 5, width = t.d.width;
  const GnUnit stride = gn_first(t, gridDim.x / ctas);
  GnUnit u = gn_first(t, blockIdx.x / ctas);
  GnShape p = gn_shape<T, VEC>(t, gn_groups(t, u), rank);
  const float count = (float)t.d.S * (float)width;
  const int stretches = ctas / t.csplit, stretch = rank / t.csplit, shift = __ffs(width) - 1;
  const bool aligned_groups = width <= 32 && (width & (width - 1)) == 0 && t.csplit == 1;
  gn_mail_init(mail);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // (the next unit's statistics, which nothing else brings nearer than HBM, come along with its values)
  constexpr int NG = GROUPED ? 1 : VEC;
  float mu_next[NG], rs_next[NG];
  const auto fetch = [&](const GnUnit& w, const GnShape& q, uint32_t after) {
    if constexpr (TMA) {
      if (tid == 0 && q.any && !mail.abort) {
        ptx::mbar_arrive_expect_tx(bar, 2 * box_bytes);
        gn_fetch_box(slots, &map_x, t, w, q, bar);
        gn_fetch_box(slots_g, &map_g, t, w, q, bar);
      }
    } else {
      gn_fetch<T, VEC, VPT>(slots, x, t, w, q, after);
      gn_fetch<T, VEC, VPT>(slots_g, g, t, w, q, after);
    }
    if (q.rows) {
      const size_t st = (size_t)w.b * t.d.G + w.slab * t.groups;
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        const int gr = GROUPED ? q.group : (q.in_slab + q.col * VEC + k) / width;
        mu_next[k] = __ldg(mean + st + gr), rs_next[k] = __ldg(rstd + st + gr);
      }
    }
  };
  fetch(u, p, 0);
  if (TMA && ctas == 1) __syncthreads();  // (the barrier is ready)
  if (ctas > 1) cluster.sync();  // everyone's boxes are ready
  for (unsigned round = 0;; ++round) {
    const int turn = round & 1;
    GnVec<VEC> vx[VPT], vg[VPT];
    const GnUnit next = gn_next(t, u, stride);
    const int slab_c = (int)u.slab * t.groups * width + p.in_slab;  // first channel of this CTA
    const float own_gamma = gamma && tid < p.channels ? __ldg(gamma + slab_c + tid) : 1.0f;  // of channel tid, for the sums
    GnVec<VEC> rs = {}, ga = {}, sum1 = gn_splat<VEC>(0.0f), sum2 = sum1;  // of dz and of dz * h
    {
      GnVec<VEC> mu = {}, be = {};
      if (p.rows) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) mu.e[k] = mu_next[k % NG], rs.e[k] = rs_next[k % NG];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          ga.e[k] = gamma ? __ldg(gamma + slab_c + p.col * VEC + k) : 1.0f;
          be.e[k] = beta ? __ldg(beta + slab_c + p.col * VEC + k) : 0.0f;
        }
      }
      uint32_t after = 0;
      if constexpr (TMA) {
        if (p.any) gn_wait_data(mail, round);
        gn_take_box(vx, slots, t, p);
        gn_take_box(vg, slots_g, t, p);
        gn_slots_read();
      } else {
        asm volatile("cp.async.wait_all;" ::: "memory");
        gn_take<T>(vx, slots, p.rows);
        gn_take<T>(vg, slots_g, p.rows);
        after = gn_after(t, vx) | gn_after(t, vg);
      }
      if (next.unit < t.units) {
        if (gn_groups(t, next) == p.groups)
          fetch(next, p, after);
        else
          fetch(next, gn_shape<T, VEC>(t, gn_groups(t, next), rank), after);
      }
      const GnVec<VEC> minus = vneg(mu);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (i >= p.rows) break;
        const GnVec<VEC> h = vmul(vadd(vx[i], minus), rs);
        vg[i] = act_bwd<ACT>(vg[i], vx[i], mu, rs, ga, be, h);  // dz
        vx[i] = h;
        sum1 = vadd(sum1, vg[i]);
        sum2 = vfma(vg[i], h, sum2);
      }
    }
    float2 acc[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) acc[k] = make_float2(sum1.e[k], sum2.e[k]);
    if (p.even) {
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        if (o < p.cols) break;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          acc[k].x += __shfl_xor_sync(~0u, acc[k].x, o);
          acc[k].y += __shfl_xor_sync(~0u, acc[k].y, o);
        }
      }
      if ((tid & 31) < p.cols) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) sm_chan[(warp * p.cols + p.col) * VEC + k] = acc[k];
      }
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) sm_chan[tid * VEC + k] = acc[k];
    }
    __syncthreads();
    const int parts = p.even ? T / 32 : p.lanes, padded = p.cols * VEC;  // rows of sums, and how far they are apart
    for (int c0 = warp * 32; c0 < p.channels; c0 += T) {  // whole warps
      const int ch = c0 + (tid & 31);
      float2 s = make_float2(0.f, 0.f);
      if (ch < p.channels) {
        s = sm_chan[ch];
        for (int q = 1; q < parts; ++q) {
          const float2 e = sm_chan[q * padded + ch];
          s.x += e.x, s.y += e.y;
        }
        if (sums) sums[((size_t)u.b * stretches + stretch) * t.d.C + slab_c + ch] = s;
        const float w = ch == tid ? own_gamma : gamma ? __ldg(gamma + slab_c + ch) : 1.0f;
        s = make_float2(w * s.x, w * s.y);
      }
      if (aligned_groups) {  // a group's channels are neighbouring lanes
#pragma unroll
        for (int o = 16; o; o >>= 1)
          if (o < width) s.x += __shfl_xor_sync(~0u, s.x, o), s.y += __shfl_xor_sync(~0u, s.y, o);
        if (dx && ch < p.channels && (ch & (width - 1)) == 0) gn_send(mail, turn, rank, ctas, ch >> shift, s);
      } else if (ch < p.channels) {
        sm_part[ch] = s;
      }
    }
    if (dx) {
      if (!aligned_groups) {
        __syncthreads();
        for (int gr = warp; gr < p.groups; gr += T / 32) {
          const int lo = max(gr * width - p.in_slab, 0), hi = min((gr + 1) * width - p.in_slab, p.channels);
          float2 s = make_float2(0.f, 0.f);
          for (int ch = lo + (tid & 31); ch < hi; ch += 32) s.x += sm_part[ch].x, s.y += sm_part[ch].y;
#pragma unroll
          for (int o = 16; o; o >>= 1) s.x += __shfl_xor_sync(~0u, s.x, o), s.y += __shfl_xor_sync(~0u, s.y, o);
          if ((tid & 31) == 0) gn_send(mail, turn, rank, ctas, gr, s);
        }
      }
      if (ctas == 1) __syncthreads();
      if (warp == 0 && ctas > 1) gn_receive(mail, turn, round, ctas, p.groups);
      if (tid < p.groups) {
        float2 s = make_float2(0.f, 0.f);
        for (int r = 0; r < ctas; ++r) s.x += mail.box[turn][r][tid].x, s.y += mail.box[turn][r][tid].y;
        sm_coef[tid] = make_float2(s.x / count, s.y / count);
      }
      __syncthreads();
      if (p.rows) {
        GnVec<VEC> c1, c2;  // minus rstd times the two means
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float2 m = sm_coef[GROUPED ? p.group : (p.in_slab + p.col * VEC + k) / width];
          c1.e[k] = -rs.e[k] * m.x, c2.e[k] = -rs.e[k] * m.y;
        }
        ga = vmul(ga, rs);
        float* to = dx + gn_base(t, u) + p.inside;
        const size_t step = (size_t)p.lanes * t.d.C;
#pragma unroll
        for (int i = 0; i < VPT; ++i, to += step) {
          if (i >= p.rows) break;
          gn_store<VEC>(to, vfma(ga, vg[i], vfma(vx[i], c2, c1)));
        }
      }
    } else {
      __syncthreads();
    }
    if (next.unit >= t.units) break;
    u = next;
    if (gn_groups(t, u) != p.groups) p = gn_shape<T, VEC>(t, gn_groups(t, u), rank);
  }
  if (TMA || ctas > 1) ptx::report_abort(&mail.abort, status, VTLB_ST_NORM_TIMEOUT);  // whichever thread's wait it was
  if (TMA && p.any) gn_last_copies(mail);
  if (ctas > 1) cluster.sync();
}

// What is known of one kernel: how many clusters of each size the GPU holds at a time (asked once: the library runs on one
// kind of GPU), and per device whether it has been allowed the most shared memory that any plan asks for.
struct GnKernelInfo {
  static constexpr int kDevices = 16;
  std::atomic<int> resident[kGnMaxCluster + 1];
  std::atomic<bool> allowed[kDevices];
};

// Launches as many clusters as the GPU holds at a time (each goes on to further units), at most one per unit.  `usual` is
// the shared memory that threads full of rows take, for which the clusters are counted whatever this call's rows.
template <typename... KArgs, typename... Args>
cudaError_t cluster_launch(vtlb_ctx* ctx, GnKernelInfo& info, void (*kern)(KArgs...), int threads, unsigned units,
                           int cluster, size_t smem, size_t usual, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute at[2];
  if (vtlb_early_on()) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    auto& dim = at[cfg.numAttrs++].val.clusterDim;
    dim.x = cluster, dim.y = 1, dim.z = 1;
  }
  cfg.attrs = at;
  cudaError_t e;
  std::atomic<bool>* allowed = ctx->device < GnKernelInfo::kDevices ? &info.allowed[ctx->device] : nullptr;
  if (!allowed || !allowed->load(std::memory_order_relaxed)) {
    if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kGnMaxSmem)) != cudaSuccess) return e;
    if (allowed) allowed->store(true, std::memory_order_relaxed);
  }
  unsigned clusters = units;
  if (units > 8) {
    int fit = info.resident[cluster].load(std::memory_order_relaxed);
    if (!fit) {
      if (cluster > 1) {
        cfg.dynamicSmemBytes = usual;
        e = cudaOccupancyMaxActiveClusters(&fit, kern, &cfg);
        cfg.dynamicSmemBytes = smem;
      } else {
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kern, threads, usual);
        fit *= ctx->sm_count;
      }
      if (e != cudaSuccess) return e;
      if (fit < 1) fit = 1;
      info.resident[cluster].store(fit, std::memory_order_relaxed);
    }
    // as few as finish in the same number of rounds: a cluster that finds no room yet would run behind all others
    const unsigned rounds = (units + fit - 1) / fit;
    clusters = (units + rounds - 1) / rounds;
  }
  cfg.gridDim = dim3(clusters * cluster);
  return cudaLaunchKernelEx(&cfg, kern, static_cast<Args&&>(args)...);
}
template <int ACT, int VEC, int VPT, bool GROUPED, bool TMA, typename... Args>
cudaError_t fwd_tile(vtlb_ctx* ctx, const GnTile& t, int cluster, Args... args) {
  static GnKernelInfo info;
  const size_t usual = (size_t)kGnFwdThreads * VPT * VEC * 4, smem = TMA ? (size_t)t.boxes * t.box_rows * t.channels * 4 : usual;
  return cluster_launch(ctx, info, gn_fwd_tile_kernel<ACT, VEC, VPT, GROUPED, TMA>, kGnFwdThreads, t.units, cluster, smem, usual, args...);
}
template <int ACT, int VEC, int VPT, bool GROUPED, bool TMA, typename... Args>
cudaError_t bwd_tile(vtlb_ctx* ctx, const GnTile& t, int cluster, Args... args) {
  static GnKernelInfo info;
  const size_t usual = (size_t)kGnBwdThreads * VPT * VEC * 8, smem = TMA ? (size_t)t.boxes * t.box_rows * t.channels * 8 : usual;
  return cluster_launch(ctx, info, gn_bwd_tile_kernel<ACT, VEC, VPT, GROUPED, TMA>, kGnBwdThreads, t.units, cluster, smem, usual, args...);
}

GnTile tile_of(const GnDims& d, const GnPlan& p, bool in_place) { return GnTile{d, p.groups, p.slabs, p.csplit, p.channels, p.rows, (unsigned)d.B * (unsigned)p.slabs, 0u,
                p.boxes, p.box_rows, in_place}; }

int check_dims(vtlb_ctx* ctx, const char* fn, int B, int S, int C, int groups, int act_kind, GnDims* d) {
  if (B <= 0 || S <= 0 || C <= 0 || groups <= 0 || C % groups)
    return vtlb_fail(ctx, VTLB_EINVAL, "%s: bad shape B=%d S=%d C=%d groups=%d", fn, B, S, C, groups);
  if (act_kind != VTLB_ACT_NONE && act_kind != VTLB_ACT_RELU && act_kind != VTLB_ACT_SILU)
    return vtlb_fail(ctx, VTLB_EINVAL, "%s: unknown activation %d", fn, act_kind);
  if (C > kGnMaxChannels) return vtlb_fail(ctx, VTLB_EINVAL, "%s: C=%d: channels go to %d", fn, C, kGnMaxChannels);
  // (CTAs, units and rows of sums are counted in 31 bits; a sample's chunks are a grid's second dimension)
  if ((long long)B * groups > INT_MAX || (long long)B * S > INT_MAX || S > 65535 * kRows)
    return vtlb_fail(ctx, VTLB_EINVAL, "%s: B=%d S=%d groups=%d: B * S and B * groups go to 2^31 - 1, S to %d", fn, B, S, groups, 65535 * kRows);
  *d = GnDims{B, S, C, groups, C / groups};
  return VTLB_OK;
}

GnGrid grid_of(const GnDims& d, int vec, int sm_count) {
  GnGrid t{d, 0, kRows, 1};
  while (t.shift < 8 && (1 << t.shift) * vec < d.C && ((1 << t.shift) < 32 || d.S * (1 << t.shift) < kRows * 8)) ++t.shift;
  // 32 pieces wide as a rule, wider where there are few rows; four rows a thread at least.
  t.across = (d.C + (vec << t.shift) - 1) / (vec << t.shift);
  const long long ctas = (long long)d.B * t.across;
  while (t.rows > 4 * (256 >> t.shift) && t.rows > 32 && ctas * ((d.S + t.rows - 1) / t.rows) < 2LL * sm_count) t.rows /= 2;
  return t;
}

int group_threads(const GnDims& d, int chunks) { return (long long)chunks * d.width > 256 ? 256 : 32; }

template <int ACT, int VEC>
int gn_forward_general(vtlb_ctx* ctx, const float* x, GnDims d, const float* gamma, const float* beta, double eps, float* y,
                       float* mean, float* rstd) {
  const GnGrid t = grid_of(d, VEC, ctx->sm_count);
  const int chunks = (d.S + t.rows - 1) / t.rows;
  const dim3 grid((unsigned)d.B * t.across, chunks);
  vtlb_workspace ws(ctx);
  void* partial = nullptr;
  if (int rc = ws.get((size_t)d.B * chunks * d.C * sizeof(double2), &partial)) return rc;
  const float* none = nullptr;
  VTLB_CUDA(ctx, vtlb_launch_early(gn_sums_kernel<ACT, false, VEC>, grid, dim3(256), 0, ctx->stream, x, none, none, none, none,
                                   none, t, (double2*)partial));
  VTLB_LAUNCHED(ctx);
  VTLB_CUDA(ctx, vtlb_launch_early(gn_groups_kernel<false>, dim3((unsigned)d.B * d.G), dim3(group_threads(d, chunks)), 0,
                                   ctx->stream, (const double2*)partial, chunks, d, x, none, eps, mean, rstd, (float2*)nullptr));
  VTLB_LAUNCHED(ctx);
  VTLB_CUDA(ctx, vtlb_launch_early(gn_apply_kernel<ACT, false, VEC>, grid, dim3(256), 0, ctx->stream, x, none, gamma, beta,
                                   (const float*)mean, (const float*)rstd, (const float2*)nullptr, t, y));
  VTLB_LAUNCHED(ctx);
  return VTLB_OK;
}

template <int ACT, int VEC>
int gn_backward_general(vtlb_ctx* ctx, const float* g, const float* x, GnDims d, const float* gamma, const float* beta,
                        const float* mean, const float* rstd, float* dx, float* dgamma, float* dbeta) {
  const GnGrid t = grid_of(d, VEC, ctx->sm_count);
  const int chunks = (d.S + t.rows - 1) / t.rows;
  const dim3 grid((unsigned)d.B * t.across, chunks);
  const size_t sums = (size_t)d.B * chunks * d.C * sizeof(double2);
  vtlb_workspace ws(ctx);
  void* scratch = nullptr;
  if (int rc = ws.get(sums + (size_t)d.B * d.G * sizeof(float2), &scratch)) return rc;
  double2* partial = (double2*)scratch;
  float2* coef = (float2*)((char*)scratch + sums);
  VTLB_CUDA(ctx, vtlb_launch_early(gn_sums_kernel<ACT, true, VEC>, grid, dim3(256), 0, ctx->stream, x, g, gamma, beta, mean,
                                   rstd, t, partial));
  VTLB_LAUNCHED(ctx);
  if (dgamma || dbeta) {
    VTLB_CUDA(ctx, vtlb_launch_early(gn_params_kernel<double2>, dim3((d.C + 7) / 8), dim3(256), 0, ctx->stream,
                                     (const double2*)partial, d.B * chunks, d.C, dgamma, dbeta));
    VTLB_LAUNCHED(ctx);
  }
  if (!dx) return VTLB_OK;
  VTLB_CUDA(ctx, vtlb_launch_early(gn_groups_kernel<true>, dim3((unsigned)d.B * d.G), dim3(group_threads(d, chunks)), 0,
                                   ctx->stream, (const double2*)partial, chunks, d, x, gamma, 0.0, (float*)nullptr,
                                   (float*)nullptr, coef));
  VTLB_LAUNCHED(ctx);
  VTLB_CUDA(ctx, vtlb_launch_early(gn_apply_kernel<ACT, true, VEC>, grid, dim3(256), 0, ctx->stream, x, g, gamma, beta, mean,
                                   rstd, (const float2*)coef, t, dx));
  VTLB_LAUNCHED(ctx);
  return VTLB_OK;
}

// Threads per row and pieces per thread, the fewest that hold it (pieces of four values, or one); false: too long a row.
bool gn_row_shape(int width, int vec, bool bwd, int* threads, int* per) {
  const int shapes[2][7][2] = {{{8, 2}, {8, 8}, {32, 4}, {32, 8}, {256, 2}, {256, 4}, {256, 8}},
                               {{8, 2}, {32, 2}, {64, 2}, {128, 2}, {256, 2}, {256, 4}, {256, 8}}};
  for (const auto& s : shapes[bwd])
    if (width <= s[0] * s[1] * vec) {
      *threads = s[0], *per = s[1];
      return true;
    }
  return false;
}

template <int ACT, int VEC>
int gn_forward_rows(vtlb_ctx* ctx, int threads, int per, const float* x, GnDims d, const float* gamma, const float* beta,
                    double eps, float* y, float* mean, float* rstd) {
  auto kern = threads == 8 ? (per == 2 ? gn_rows_fwd_kernel<ACT, VEC, 8, 2> : gn_rows_fwd_kernel<ACT, VEC, 8, 8>)
              : threads == 32 ? (per == 4 ? gn_rows_fwd_kernel<ACT, VEC, 32, 4> : gn_rows_fwd_kernel<ACT, VEC, 32, 8>)
              : per == 2      ? gn_rows_fwd_kernel<ACT, VEC, 256, 2>
              : per == 4      ? gn_rows_fwd_kernel<ACT, VEC, 256, 4>
                              : gn_rows_fwd_kernel<ACT, VEC, 256, 8>;
  const int places = kGnRowThreads / threads;
  const size_t ctas = ((size_t)d.B * d.G + places - 1) / places;
  VTLB_CUDA(ctx, vtlb_launch_early(kern, dim3((unsigned)ctas), dim3(kGnRowThreads), 0, ctx->stream, x, gamma, beta, d, (float)eps, 1.0 / (double)d.width, y, mean, rstd));
  VTLB_LAUNCHED(ctx);
  return VTLB_OK;
}

template <int ACT, int VEC>
int gn_backward_rows(vtlb_ctx* ctx, int threads, int per, const float* g, const float* x, GnDims d, const float* gamma,
                     const float* beta, const float* mean, const float* rstd, float* dx, float* dgamma, float* dbeta) {
  auto kern = threads == 8 ? gn_rows_bwd_kernel<ACT, VEC, 8, 2>
              : threads == 32  ? gn_rows_bwd_kernel<ACT, VEC, 32, 2>
              : threads == 64  ? gn_rows_bwd_kernel<ACT, VEC, 64, 2>
              : threads == 128 ? gn_rows_bwd_kernel<ACT, VEC, 128, 2>
              : per == 2       ? gn_rows_bwd_kernel<ACT, VEC, 256, 2>
              : per == 4       ? gn_rows_bwd_kernel<ACT, VEC, 256, 4>
                               : gn_rows_bwd_kernel<ACT, VEC, 256, 8>;
  // Up to 64 rows to a place, but eight CTAs per SM first; four, where that takes fewer than sixteen rows each, whose
  // sums are a twelfth of the bytes (10000 x 4096: 101 us with sixteen, 110 with eight).
  const int places = kGnRowThreads / threads;
  const long long steps = ((long long)d.B + places - 1) / places;
  const long long fill = steps * d.G / ((long long)ctx->sm_count * 4);  // rows to a place with four CTAs per SM
  const long long each = fill < 1 ? 1 : fill <= 16 ? fill : fill <= 32 ? 16 : fill <= 128 ? fill / 2 : 64;
  const long long chunks = (steps + each - 1) / each;
  vtlb_workspace ws(ctx);
  void* sums = nullptr;
  if (dgamma || dbeta)
    if (int rc = ws.get((size_t)chunks * d.C * sizeof(float2), &sums)) return rc;
  VTLB_CUDA(ctx, vtlb_launch_early(kern, dim3((unsigned)(chunks * d.G)), dim3(kGnRowThreads), 0, ctx->stream, g, x, gamma, beta, mean,
                                   rstd, d, (int)each, dx, (float2*)sums));
  VTLB_LAUNCHED(ctx);
  if (!sums) return VTLB_OK;
  VTLB_CUDA(ctx, vtlb_launch_early(gn_params_kernel<float2>, dim3((d.C + 7) / 8), dim3(256), 0, ctx->stream, (const float2*)sums,
                                   (int)chunks, d.C, dgamma, dbeta));
  VTLB_LAUNCHED(ctx);
  return VTLB_OK;
}

template <int ACT>
int gn_forward(vtlb_ctx* ctx, const float* x, GnDims d, const float* gamma, const float* beta, double eps, float* y,
               float* mean, float* rstd) {
  if (d.S == 1 && (eps == 0.0 || (eps >= 1e-30 && eps <= 1e30))) {  // (eps as f32; 500000 rows of 64 40 us, in f64 44)
    const bool vec = d.width % 4 == 0 && vtlb_aligned16(x) && vtlb_aligned16(y) && vtlb_aligned16(gamma) && vtlb_aligned16(beta);
    int threads, per;
    if (gn_row_shape(d.width, vec ? 4 : 1, false, &threads, &per))
      return vec ? gn_forward_rows<ACT, 4>(ctx, threads, per, x, d, gamma, beta, eps, y, mean, rstd)
                 : gn_forward_rows<ACT, 1>(ctx, threads, per, x, d, gamma, beta, eps, y, mean, rstd);
  }
  const GnPlan plan = gn_plan(d.B, d.S, d.C, d.G, vtlb_aligned16(x) && vtlb_aligned16(y), kGnFwdThreads, 4, 16, ctx->sm_count);
  if (plan.on_chip) {
    const GnTile t = tile_of(d, plan, x == y);
    const int cluster = plan.csplit * plan.rsplit;
    const bool grouped = d.width % 4 == 0;
    CUtensorMap map = {};
    if (plan.tma)
      if (int rc = gemm::encode_tmap_3d_f32_plain(ctx, &map, x, d.C, d.S, d.B, plan.channels, plan.box_rows)) return rc;
#define VTLB_GN_FWD(VEC, VPT, GROUPED, TMA) \
  fwd_tile<ACT, VEC, VPT, GROUPED, TMA>(ctx, t, cluster, map, x, gamma, beta, t, eps, y, mean, rstd, ctx->d_status)
#define VTLB_GN_FWD_VPT(VPT)                                                      \
  case VPT:                                                                       \
    VTLB_CUDA(ctx, plan.vec == 1 ? VTLB_GN_FWD(1, VPT, true, false)               \
                   : !plan.tma   ? VTLB_GN_FWD(4, VPT, false, false)              \
                   : grouped     ? VTLB_GN_FWD(4, VPT, true, true)                \
                                 : VTLB_GN_FWD(4, VPT, false, true));             \
    break
    switch (plan.vpt) {
      VTLB_GN_FWD_VPT(1);
      VTLB_GN_FWD_VPT(4);
      VTLB_GN_FWD_VPT(16);
    }
#undef VTLB_GN_FWD_VPT
#undef VTLB_GN_FWD
    VTLB_LAUNCHED(ctx);
    return VTLB_OK;
  }
  return plan.vec == 4 ? gn_forward_general<ACT, 4>(ctx, x, d, gamma, beta, eps, y, mean, rstd)
                       : gn_forward_general<ACT, 1>(ctx, x, d, gamma, beta, eps, y, mean, rstd);
}

template <int ACT>
int gn_backward(vtlb_ctx* ctx, const float* g, const float* x, GnDims d, const float* gamma, const float* beta,
                const float* mean, const float* rstd, float* dx, float* dgamma, float* dbeta) {
  const bool aligned = vtlb_aligned16(x) && vtlb_aligned16(g) && vtlb_aligned16(dx);
  if (d.S == 1) {
    const bool vec = d.width % 4 == 0 && aligned && vtlb_aligned16(gamma) && vtlb_aligned16(beta);
    int threads, per;
    if (gn_row_shape(d.width, vec ? 4 : 1, true, &threads, &per))
      return vec ? gn_backward_rows<ACT, 4>(ctx, threads, per, g, x, d, gamma, beta, mean, rstd, dx, dgamma, dbeta)
                 : gn_backward_rows<ACT, 1>(ctx, threads, per, g, x, d, gamma, beta, mean, rstd, dx, dgamma, dbeta);
  }
  const GnPlan plan = gn_plan(d.B, d.S, d.C, d.G, aligned, kGnBwdThreads, 4, 8, ctx->sm_count);
  vtlb_workspace ws(ctx);
  void* scratch = nullptr;
  if (plan.on_chip) {
    const GnTile t = tile_of(d, plan, false);
    const int cluster = plan.csplit * plan.rsplit;
    const int rows = d.B * plan.rsplit;
    if (dgamma || dbeta)
      if (int rc = ws.get((size_t)rows * d.C * sizeof(float2), &scratch)) return rc;
    float2* sums = (float2*)scratch;
    const bool grouped = d.width % 4 == 0;
    CUtensorMap map_g = {}, map_x = {};
    if (plan.tma) {
      if (int rc = gemm::encode_tmap_3d_f32_plain(ctx, &map_g, g, d.C, d.S, d.B, plan.channels, plan.box_rows)) return rc;
      if (int rc = gemm::encode_tmap_3d_f32_plain(ctx, &map_x, x, d.C, d.S, d.B, plan.channels, plan.box_rows)) return rc;
    }
#define VTLB_GN_BWD(VEC, VPT, GROUPED, TMA)                                                                        \
  bwd_tile<ACT, VEC, VPT, GROUPED, TMA>(ctx, t, cluster, map_g, map_x, g, x, gamma, beta, mean, rstd, t, dx, sums, \
                                        ctx->d_status)
#define VTLB_GN_BWD_VPT(VPT)                                                      \
  case VPT:                                                                       \
    VTLB_CUDA(ctx, plan.vec == 1 ? VTLB_GN_BWD(1, VPT, true, false)               \
                   : !plan.tma   ? VTLB_GN_BWD(4, VPT, false, false)              \
                   : grouped     ? VTLB_GN_BWD(4, VPT, true, true)                \
                                 : VTLB_GN_BWD(4, VPT, false, true));             \
    break
    switch (plan.vpt) {
      VTLB_GN_BWD_VPT(1);
      VTLB_GN_BWD_VPT(4);
      VTLB_GN_BWD_VPT(8);
    }
#undef VTLB_GN_BWD_VPT
#undef VTLB_GN_BWD
    VTLB_LAUNCHED(ctx);
    if (sums) {
      VTLB_CUDA(ctx, vtlb_launch_early(gn_params_kernel<float2>, dim3((d.C + 7) / 8), dim3(256), 0, ctx->stream,
                                       (const float2*)sums, rows, d.C, dgamma, dbeta));
      VTLB_LAUNCHED(ctx);
    }
    return VTLB_OK;
  }
  return plan.vec == 4 ? gn_backward_general<ACT, 4>(ctx, g, x, d, gamma, beta, mean, rstd, dx, dgamma, dbeta)
                       : gn_backward_general<ACT, 1>(ctx, g, x, d, gamma, beta, mean, rstd, dx, dgamma, dbeta);
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
