// Dropout whose mask is never stored: y_i = x_i / (1 - p) where the generator's word i is at least p * 2^32, else 0
// (philox.cuh).  The gradient of it is the same map on the upstream gradient, so forward and backward share a kernel.
#include "philox.cuh"

namespace {

__global__ void __launch_bounds__(256) dropout_kernel(const float* x, float* y, size_t n, int vec, vtlb_mask m) {
  const size_t tid = blockIdx.x * (size_t)blockDim.x + threadIdx.x, stride = (size_t)gridDim.x * blockDim.x;
  const size_t n4 = n / 4;
  if (vec) {
    for (size_t i = tid; i < n4; i += stride)
      reinterpret_cast<float4*>(y)[i] = vtlb_drop4(m, i, reinterpret_cast<const float4*>(x)[i]);
  } else {
    for (size_t i = tid; i < n4; i += stride) {
      const float4 v = vtlb_drop4(m, i, make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]));
      y[4 * i] = v.x, y[4 * i + 1] = v.y, y[4 * i + 2] = v.z, y[4 * i + 3] = v.w;
    }
  }
  if (tid < n - 4 * n4) {
    const uint4 r = vtlb_philox(m, n4);
    const uint32_t w = tid == 0 ? r.x : tid == 1 ? r.y : r.z;
    y[4 * n4 + tid] = vtlb_drop(m, w, x[4 * n4 + tid]);
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
  const size_t want = (n / 4 + 255) / 256, cap = (size_t)ctx->sm_count * 16;
  const int grid = (int)(want > cap ? cap : want < 1 ? 1 : want);
  const int vec = vtlb_aligned16(d_x) && vtlb_aligned16(d_y);
  dropout_kernel<<<grid, 256, 0, ctx->stream>>>((const float*)d_x, (float*)d_y, n, vec, m);
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
