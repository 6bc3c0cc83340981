// Dropout whose mask is never stored: y_i = x_i / (1 - p) where the generator's word i is at least p * 2^32, else 0
// (philox.cuh).  The gradient of it is the same map on the upstream gradient, so forward and backward share a kernel.
#include "philox.cuh"

namespace {

// U blocks of four elements per thread, loaded before any is worked on.  VEC: both arrays are 16-byte aligned.  Bound by
// HBM, 8 bytes per element: 16384 x 4096 in 78 to 84 us, 6.4 to 6.9 TB/s, a plain copy's rate (the twenty wide products
// of a block of the mask take a quarter of that time on the integer pipe).  64 x 256: 4.2 us, the host's call.
template <bool VEC, int U>
__global__ void __launch_bounds__(256) dropout_kernel(const float* x, float* y, size_t n, vtlb_mask m) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early: the kernel in front is done from here on
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const size_t n4 = n / 4, first = blockIdx.x * (size_t)(256 * U) + threadIdx.x;
  float4 v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const size_t i = first + u * 256;
    v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < n4)
      v[u] = VEC ? reinterpret_cast<const float4*>(x)[i] : make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const size_t i = first + u * 256;
    if (i >= n4) break;
    const float4 o = vtlb_drop4(m, i, v[u]);
    if (VEC)
      reinterpret_cast<float4*>(y)[i] = o;
    else
      y[4 * i] = o.x, y[4 * i + 1] = o.y, y[4 * i + 2] = o.z, y[4 * i + 3] = o.w;
  }
  if (blockIdx.x == 0 && threadIdx.x < n - 4 * n4) {
    const uint4 r = vtlb_philox(m, n4);
    const uint32_t w = threadIdx.x == 0 ? r.x : threadIdx.x == 1 ? r.y : r.z;
    y[4 * n4 + threadIdx.x] = vtlb_drop(m, w, x[4 * n4 + threadIdx.x]);
  }
}

int dropout(vtlb_ctx* ctx, const char* fn, const void* d_x, void* d_y, size_t n, double p, uint64_t seed, uint64_t step) {
  if (!(p >= 0.0 && p <= 1.0)) return vtlb_fail(ctx, VTLB_EINVAL, "%s: p must be in [0, 1]", fn);
  if (n == 0) return VTLB_OK;
  if (!d_x || !d_y) return vtlb_fail(ctx, VTLB_EINVAL, "%s: null pointer", fn);
  if (d_x != d_y && vtlb_overlap(d_x, n, d_y, n))
    return vtlb_fail(ctx, VTLB_EINVAL, "%s: input and output overlap in part", fn);
  const vtlb_mask m = vtlb_make_mask(p, seed, step);
  if (!m.any) {
    if (d_x != d_y) VTLB_CUDA(ctx, cudaMemcpyAsync(d_y, d_x, n * sizeof(float), cudaMemcpyDeviceToDevice, ctx->stream));
    return VTLB_OK;
  }
  const bool vec = vtlb_aligned16(d_x) && vtlb_aligned16(d_y);
  // Four blocks per thread (16384 x 4096 elements: 78 us, two 84, one 87) where that still leaves work for every SM.
  const int U = n >= (size_t)ctx->sm_count * 4 * 256 * 4 * 2 ? 4 : 1;
  const size_t ctas = (n + 1024 * U - 1) / (1024 * U);
  if (ctas > 0x7fffffffu) return vtlb_fail(ctx, VTLB_EINVAL, "%s: more than 2^41 elements", fn);
  auto kern = U == 4 ? (vec ? dropout_kernel<true, 4> : dropout_kernel<false, 4>)
                     : (vec ? dropout_kernel<true, 1> : dropout_kernel<false, 1>);
  VTLB_CUDA(ctx, vtlb_launch_early(kern, dim3((unsigned)ctas), dim3(256), 0, ctx->stream, (const float*)d_x, (float*)d_y, n, m));
  VTLB_LAUNCHED(ctx);
  return VTLB_OK;
}

}  // namespace

VTLB_API int vtlb_dropout_fwd_f32(vtlb_ctx* ctx, const void* d_x, void* d_y, size_t n, double p, uint64_t seed,
                                  uint64_t step) {
  VTLB_ENTER(ctx);
  return dropout(ctx, "vtlb_dropout_fwd_f32", d_x, d_y, n, p, seed, step);
}

VTLB_API int vtlb_dropout_bwd_f32(vtlb_ctx* ctx, const void* d_g, void* d_dx, size_t n, double p, uint64_t seed,
                                  uint64_t step) {
  VTLB_ENTER(ctx);
  return dropout(ctx, "vtlb_dropout_bwd_f32", d_g, d_dx, n, p, seed, step);
}
