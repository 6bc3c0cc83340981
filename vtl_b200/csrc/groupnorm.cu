// Group norm with an activation, channels last: x[B, S, C] (S positions: H * W of a feature map, the length of a
// sequence, 1 for plain features), C channels in `groups` equal groups.  Per sample and group, over S * C/groups values,
//   h = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps) (biased variance),  z = gamma_c * h + beta_c,  y = act(z).
// Backward, with dz = g * act'(z) and n = S * C/groups:
//   dgamma_c = sum over samples and positions of dz * h,   dbeta_c = sum of dz,
//   dx = rstd * (gamma_c * dz - (sum gamma dz) / n - h * (sum gamma dz h) / n), the sums over the group.
#include <cooperative_groups.h>

#include "common.cuh"
#include "groupnorm_plan.h"

namespace {

struct GnDims {
  int B, S, C, G, width;  // width = C / G
};

// 1 / (1 + exp(-z)) within 7 half steps: expf 4, the sum 1, the approximate division (1 ulp) 2.  IEEE division would
// take some eight instructions more per element, a fifth of the forward kernel's.  Below -87.3, where the sum passes
// 2^126, the division gives 0 (the logistic function is under 1.2e-38 there).
__device__ __forceinline__ float logistic(float z) { return __fdividef(1.0f, 1.0f + expf(-z)); }

template <int ACT>
__device__ __forceinline__ float act(float z) {
  if (ACT == VTLB_ACT_RELU) return z < 0.0f ? 0.0f : z;
  if (ACT == VTLB_ACT_SILU) return z * logistic(z);
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
  const float s = logistic(z);
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

// ---------------------------------------------------------------- groups that fit the registers of a cluster
// x is read once: it stays in registers between the sums and the result (groupnorm_plan.h).  Bound by HBM, 8 bytes per
// element forward, 12 backward.
struct GnTile {
  GnDims d;
  int groups, slabs, csplit, channels, rows;
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

// Where this CTA and thread stand.
struct GnPlace {
  int b, grp0, groups;  // sample, first group of the slab, groups in it
  int c0, channels;     // first channel and channels of this CTA
  int in_slab;          // c0 minus the slab's first channel
  int cols, lanes;      // pieces of VEC channels, rows per step
  int col, lane;        // this thread's
  int r0, r1;           // rows of this CTA
  bool on;
  bool even;            // pieces of a row fill a warp evenly: cols is a power of two up to 32
};
template <int VEC>
__device__ __forceinline__ GnPlace gn_place(const GnTile& t, int rank, int cluster) {
  GnPlace p;
  const unsigned unit = blockIdx.x / cluster;
  p.b = (int)(unit / t.slabs);
  const int slab = (int)(unit % t.slabs);
  p.grp0 = slab * t.groups;
  p.groups = min(t.groups, t.d.G - p.grp0);
  p.in_slab = (rank % t.csplit) * t.channels;
  p.c0 = p.grp0 * t.d.width + p.in_slab;
  p.channels = min(t.channels, p.groups * t.d.width - p.in_slab);
  p.cols = p.channels / VEC;
  p.lanes = kGnThreads / p.cols;
  p.col = threadIdx.x % p.cols;
  p.lane = threadIdx.x / p.cols;
  p.r0 = min(t.d.S, (rank / t.csplit) * t.rows);
  p.r1 = min(t.d.S, p.r0 + t.rows);
  p.on = p.lane < p.lanes;
  p.even = p.cols <= 32 && (p.cols & (p.cols - 1)) == 0;
  return p;
}

template <int ACT, int VEC, int VPT, bool GROUPED>
__global__ void __launch_bounds__(kGnThreads, VPT > 8 ? 1024 / kGnThreads / 2 : 1024 / kGnThreads) gn_fwd_tile_kernel(const float* x, const float* gamma, const float* beta,
                                                                 GnTile t, double eps, float* y, float* mean_out,
                                                                 float* rstd_out) {
  namespace cg = cooperative_groups;
  constexpr int PAIRS = GROUPED ? 1 : VEC;  // GROUPED: the channels of a thread's piece are all of one group
  __shared__ double2 sm_pair[kGnThreads * PAIRS];
  __shared__ double2 sm_sum[kGnMaxGroups];
  __shared__ float2 sm_stat[kGnMaxGroups];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const GnPlace p = gn_place<VEC>(t, rank, ctas);
  const int tid = threadIdx.x, warp = tid >> 5, width = t.d.width;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early: the kernel in front is done from here on
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const size_t base = ((size_t)p.b * t.d.S + p.r0 + p.lane) * t.d.C + p.c0 + (size_t)p.col * VEC;
  const size_t step = (size_t)p.lanes * t.d.C;
  const int rows = p.on ? min(VPT, max(0, (p.r1 - p.r0 - p.lane + p.lanes - 1) / p.lanes)) : 0;  // of this thread
  GnVec<VEC> v[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i < rows) {
      v[i] = gn_load<VEC>(x + base + i * step);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) v[i].e[k] = 0.0f;
    }
  }
  // A thread's own mean K and squared distances from it in f32, then sums of x and x^2 in f64 from them: the variance
  // loses 2^-53 of the mean square, not 2^-24, and few instructions are f64.
  constexpr int PER = VEC / PAIRS;  // channels per pair
  double2 acc[PAIRS];
#pragma unroll
  for (int q = 0; q < PAIRS; ++q) {
    const float n = (float)(rows * PER);
    float sum = 0.0f, dist = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int k = 0; k < PER; ++k) sum += v[i].e[q * PER + k];
    const float mean = rows ? __fdividef(sum, n) : 0.0f;  // any value near the mean serves
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (i < rows) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const float e = v[i].e[q * PER + k] - mean;
          dist = fmaf(e, e, dist);
        }
      }
    const double nm = (double)n * (double)mean;
    acc[q] = make_double2(nm, fma(nm, (double)mean, (double)dist));
  }
  const int cq = width / PER;  // pairs per group and row
  if (p.even && (PAIRS == 1) && (cq & (cq - 1)) == 0 && cq <= p.cols) {
    // lanes of a warp that hold one group: the other rows' (steps of cols), then the other pieces of its channels
    for (int o = 16; o; o >>= 1) {
      if (o >= p.cols || o < cq) {
        acc[0].x += __shfl_xor_sync(~0u, acc[0].x, o);
        acc[0].y += __shfl_xor_sync(~0u, acc[0].y, o);
      }
    }
    const int lane = tid & 31;
    if (lane < p.cols && lane % cq == 0) sm_pair[warp * p.groups + lane / cq] = acc[0];
    __syncthreads();
    if (tid < p.groups) {
      double2 s = sm_pair[tid];
#pragma unroll
      for (int w = 1; w < kGnThreads / 32; ++w) s.x += sm_pair[w * p.groups + tid].x, s.y += sm_pair[w * p.groups + tid].y;
      sm_sum[tid] = s;
    }
  } else {
#pragma unroll
    for (int q = 0; q < PAIRS; ++q) sm_pair[tid * PAIRS + q] = acc[q];
    __syncthreads();
    // one warp per group of the slab: the pairs of its channels in this CTA, all rows
    for (int g = warp; g < p.groups; g += kGnThreads / 32) {
      const int lo = max(g * width - p.in_slab, 0) / PER, hi = min((g + 1) * width - p.in_slab, p.channels) / PER;
      double2 s = make_double2(0.0, 0.0);
      const int n = hi > lo ? hi - lo : 0, entries = p.channels / PER;
      for (int i = tid & 31; i < n * p.lanes; i += 32) {
        const double2 e = sm_pair[(i / n) * entries + lo + i % n];
        s.x += e.x, s.y += e.y;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) s.x += __shfl_xor_sync(~0u, s.x, o), s.y += __shfl_xor_sync(~0u, s.y, o);
      if ((tid & 31) == 0) sm_sum[g] = s;
    }
  }
  if (ctas > 1) cluster.sync(); else __syncthreads();
  if (tid < p.groups) {
    double2 s = make_double2(0.0, 0.0);
    for (int r = 0; r < ctas; ++r) {
      const double2 e = *cluster.map_shared_rank(&sm_sum[tid], r);
      s.x += e.x, s.y += e.y;
    }
    const double n = (double)t.d.S * width, mu = s.x / n, var = s.y / n - mu * mu;
    const float2 st = make_float2((float)mu, (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + eps)));
    sm_stat[tid] = st;
    if (rank == 0) {
      const size_t k = (size_t)p.b * t.d.G + p.grp0 + tid;
      mean_out[k] = st.x;
      rstd_out[k] = st.y;
    }
  }
  if (ctas > 1) cluster.sync(); else __syncthreads();  // (and no CTA leaves while another reads its sums)
  if (!p.on) return;
  float mu[VEC], a[VEC], be[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const int c = p.col * VEC + k;
    const float2 st = sm_stat[(p.in_slab + (GROUPED ? p.col * VEC : c)) / width];
    mu[k] = st.x;
    a[k] = gamma ? st.y * __ldg(gamma + p.c0 + c) : st.y;
    be[k] = beta ? __ldg(beta + p.c0 + c) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i >= rows) break;
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[i].e[k] = act<ACT>(fmaf(__fsub_rn(v[i].e[k], mu[k]), a[k], be[k]));
    gn_store<VEC>(y + base + i * step, v[i]);
  }
}

// Backward.  The channel sums of each CTA go to `sums` [B * rsplit][C] (dz * h, dz) for gn_params_kernel.
template <int ACT, int VEC, int VPT>
__global__ void __launch_bounds__(kGnThreads, VPT > 4 ? 1024 / kGnThreads / 2 : 1024 / kGnThreads) gn_bwd_tile_kernel(const float* g, const float* x, const float* gamma,
                                                                 const float* beta, const float* mean, const float* rstd,
                                                                 GnTile t, float* dx, float2* sums) {
  namespace cg = cooperative_groups;
  __shared__ float2 sm_part[kGnThreads * VEC];  // [lane][channel]
  __shared__ float2 sm_chan[kGnThreads * VEC];
  __shared__ float2 sm_sum[kGnMaxGroups];
  __shared__ float2 sm_coef[kGnMaxGroups];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const GnPlace p = gn_place<VEC>(t, rank, ctas);
  const int tid = threadIdx.x, warp = tid >> 5, width = t.d.width;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const size_t base = ((size_t)p.b * t.d.S + p.r0 + p.lane) * t.d.C + p.c0 + (size_t)p.col * VEC;
  const size_t step = (size_t)p.lanes * t.d.C;
  const int rows = p.on ? min(VPT, max(0, (p.r1 - p.r0 - p.lane + p.lanes - 1) / p.lanes)) : 0;
  GnVec<VEC> vx[VPT], vg[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i < rows) {
      vx[i] = gn_load<VEC>(x + base + i * step);
      vg[i] = gn_load<VEC>(g + base + i * step);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; ++k) vx[i].e[k] = vg[i].e[k] = 0.0f;
    }
  }
  float mu[VEC], rs[VEC], ga[VEC], be[VEC];
  if (p.on) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int c = p.col * VEC + k;
      const size_t st = (size_t)p.b * t.d.G + p.grp0 + (p.in_slab + c) / width;
      mu[k] = __ldg(mean + st), rs[k] = __ldg(rstd + st);
      ga[k] = gamma ? __ldg(gamma + p.c0 + c) : 1.0f;
      be[k] = beta ? __ldg(beta + p.c0 + c) : 0.0f;
    }
  }
  float2 acc[VEC] = {};
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i >= rows) break;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const float h = __fmul_rn(__fsub_rn(vx[i].e[k], mu[k]), rs[k]);
      const float dz = act_bwd<ACT>(vg[i].e[k], vx[i].e[k], mu[k], rs[k], ga[k], be[k], h);
      acc[k].x = fmaf(dz, h, acc[k].x);
      acc[k].y += dz;
      vx[i].e[k] = h, vg[i].e[k] = dz;  // what dx is made of
    }
  }
  int parts;  // rows of partial sums per channel in sm_chan
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
    parts = kGnThreads / 32;
    if ((tid & 31) < p.cols) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) sm_chan[warp * p.channels + p.col * VEC + k] = acc[k];
    }
  } else {
    if (p.on) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) sm_part[p.lane * p.channels + p.col * VEC + k] = acc[k];
    }
    __syncthreads();
    parts = max(1, min(kGnThreads / p.channels, p.lanes));
    for (int i = tid; i < parts * p.channels; i += kGnThreads) {
      const int part = i / p.channels, c = i % p.channels;
      float2 s = make_float2(0.f, 0.f);
      for (int l = part; l < p.lanes; l += parts) {
        const float2 e = sm_part[l * p.channels + c];
        s.x += e.x, s.y += e.y;
      }
      sm_chan[i] = s;
    }
  }
  __syncthreads();
  for (int c = tid; c < p.channels; c += kGnThreads) {
    float2 s = sm_chan[c];
    for (int q = 1; q < parts; ++q) {
      const float2 e = sm_chan[q * p.channels + c];
      s.x += e.x, s.y += e.y;
    }
    if (sums) sums[((size_t)p.b * (ctas / t.csplit) + rank / t.csplit) * t.d.C + p.c0 + c] = s;
    const float w = gamma ? __ldg(gamma + p.c0 + c) : 1.0f;
    sm_part[c] = make_float2(w * s.x, w * s.y);
  }
  if (!dx) return;  // (all CTAs of the cluster alike: nobody reads another's shared memory)
  __syncthreads();
  for (int gr = warp; gr < p.groups; gr += kGnThreads / 32) {
    const int lo = max(gr * width - p.in_slab, 0), hi = min((gr + 1) * width - p.in_slab, p.channels);
    float2 s = make_float2(0.f, 0.f);
    for (int c = lo + (tid & 31); c < hi; c += 32) s.x += sm_part[c].x, s.y += sm_part[c].y;
#pragma unroll
    for (int o = 16; o; o >>= 1) s.x += __shfl_xor_sync(~0u, s.x, o), s.y += __shfl_xor_sync(~0u, s.y, o);
    if ((tid & 31) == 0) sm_sum[gr] = s;
  }
  if (ctas > 1) cluster.sync(); else __syncthreads();
  if (tid < p.groups) {
    float2 s = make_float2(0.f, 0.f);
    for (int r = 0; r < ctas; ++r) {
      const float2 e = *cluster.map_shared_rank(&sm_sum[tid], r);
      s.x += e.x, s.y += e.y;
    }
    const float n = (float)t.d.S * (float)width;
    sm_coef[tid] = make_float2(s.x / n, s.y / n);
  }
  if (ctas > 1) cluster.sync(); else __syncthreads();
  if (!p.on) return;
  float2 cf[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) cf[k] = sm_coef[(p.in_slab + p.col * VEC + k) / width];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i >= rows) break;
#pragma unroll
    for (int k = 0; k < VEC; ++k) vx[i].e[k] = rs[k] * (ga[k] * vg[i].e[k] - cf[k].y - vx[i].e[k] * cf[k].x);
    gn_store<VEC>(dx + base + i * step, vx[i]);
  }
}

// dgamma and dbeta from the channel sums: 32 channels and eight stretches of rows per CTA.
__global__ void __launch_bounds__(256) gn_params_tile_kernel(const float2* sums, int rows, int C, float* dgamma, float* dbeta) {
  __shared__ double2 sm[8][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  double2 s = make_double2(0.0, 0.0);
  if (c < C) {
#pragma unroll 8
    for (int r = part; r < rows; r += 8) {
      const float2 e = sums[(size_t)r * C + c];
      s.x += (double)e.x, s.y += (double)e.y;
    }
  }
  sm[part][lane] = s;
  __syncthreads();
  if (part || c >= C) return;
  for (int q = 1; q < 8; ++q) s.x += sm[q][lane].x, s.y += sm[q][lane].y;
  if (dgamma) dgamma[c] = (float)s.x;
  if (dbeta) dbeta[c] = (float)s.y;
}

template <typename... KArgs, typename... Args>
cudaError_t cluster_launch(vtlb_ctx* ctx, void (*kern)(KArgs...), unsigned grid, int cluster, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kGnThreads);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<Args&&>(args)...);
}

GnTile tile_of(const GnDims& d, const GnPlan& p) { return GnTile{d, p.groups, p.slabs, p.csplit, p.channels, p.rows}; }

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
  const GnPlan plan = gn_plan(d.B, d.S, d.C, d.G, vtlb_aligned16(x) && vtlb_aligned16(y), 8, 16, ctx->sm_count);
  if (plan.on_chip) {
    const GnTile t = tile_of(d, plan);
    const int cluster = plan.csplit * plan.rsplit;
    const unsigned grid = (unsigned)((size_t)d.B * plan.slabs * cluster);
    const bool grouped = plan.vec == 1 || d.width % 4 == 0;
#define VTLB_GN_FWD(VEC, VPT, GROUPED) \
  cluster_launch(ctx, gn_fwd_tile_kernel<ACT, VEC, VPT, GROUPED>, grid, cluster, x, gamma, beta, t, eps, y, mean, rstd)
#define VTLB_GN_FWD_VPT(VPT) \
  case VPT:                  \
    VTLB_CUDA(ctx, plan.vec == 1 ? VTLB_GN_FWD(1, VPT, true) : grouped ? VTLB_GN_FWD(4, VPT, true) : VTLB_GN_FWD(4, VPT, false)); \
    break
    switch (plan.vpt) {
      VTLB_GN_FWD_VPT(1);
      VTLB_GN_FWD_VPT(2);
      VTLB_GN_FWD_VPT(4);
      VTLB_GN_FWD_VPT(8);
      VTLB_GN_FWD_VPT(16);
    }
#undef VTLB_GN_FWD_VPT
#undef VTLB_GN_FWD
    VTLB_LAUNCHED(ctx);
    return VTLB_OK;
  }
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
  const bool aligned = vtlb_aligned16(x) && vtlb_aligned16(g) && vtlb_aligned16(dx);
  const GnPlan plan = gn_plan(d.B, d.S, d.C, d.G, aligned, 4, 8, ctx->sm_count);
  vtlb_workspace ws(ctx);
  void* scratch = nullptr;
  if (plan.on_chip) {
    const GnTile t = tile_of(d, plan);
    const int cluster = plan.csplit * plan.rsplit;
    const unsigned grid = (unsigned)((size_t)d.B * plan.slabs * cluster);
    const int rows = d.B * plan.rsplit;
    if (dgamma || dbeta)
      if (int rc = ws.get((size_t)rows * d.C * sizeof(float2), &scratch)) return rc;
    float2* sums = (float2*)scratch;
#define VTLB_GN_BWD(VEC, VPT) \
  cluster_launch(ctx, gn_bwd_tile_kernel<ACT, VEC, VPT>, grid, cluster, g, x, gamma, beta, mean, rstd, t, dx, sums)
#define VTLB_GN_BWD_VPT(VPT) \
  case VPT:                  \
    VTLB_CUDA(ctx, plan.vec == 1 ? VTLB_GN_BWD(1, VPT) : VTLB_GN_BWD(4, VPT)); \
    break
    switch (plan.vpt) {
      VTLB_GN_BWD_VPT(1);
      VTLB_GN_BWD_VPT(2);
      VTLB_GN_BWD_VPT(4);
      VTLB_GN_BWD_VPT(8);
    }
#undef VTLB_GN_BWD_VPT
#undef VTLB_GN_BWD
    VTLB_LAUNCHED(ctx);
    if (sums) {
      VTLB_CUDA(ctx, vtlb_launch_early(gn_params_tile_kernel, dim3((d.C + 31) / 32), dim3(256), 0, ctx->stream,
                                       (const float2*)sums, rows, d.C, dgamma, dbeta));
      VTLB_LAUNCHED(ctx);
    }
    return VTLB_OK;
  }
  const int chunks = (d.S + kRows - 1) / kRows;
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
