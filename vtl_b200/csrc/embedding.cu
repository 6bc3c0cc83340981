// Embedding: y[j, :] = scale * W[ids[j], :], with or without dropout on the result (philox.cuh; the mask's element is
// the flat index in y), and its gradient dW[v, :] = scale * sum of the (masked) g[j, :] over the positions j of v.
// A position whose id lies outside the table (padding) gives a row of zeros and takes part in no gradient.
#include "philox.cuh"

namespace {

// one thread per four consecutive elements of y
template <bool DROP>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(const float* __restrict__ W, int V, uint32_t D,
                                                            const int32_t* __restrict__ ids, size_t total, float scale,
                                                            float* __restrict__ y, vtlb_mask m, uint32_t* bad) {
  for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; 4 * i < total; i += (size_t)gridDim.x * blockDim.x) {
    uint4 r = make_uint4(0, 0, 0, 0);
    if (DROP) r = vtlb_philox(m, i);
    const uint32_t word[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const size_t e = 4 * i + k;
      if (e >= total) break;
      const size_t j = e / D;
      const int id = ids[j];
      const bool in = id >= 0 && id < V;
      if (!in && bad) atomicOr(bad, 1u);
      float v = in ? __fmul_rn(W[(size_t)id * D + (e - j * D)], scale) : 0.0f;
      if (DROP) v = vtlb_drop(m, word[k], v);
      y[e] = v;
    }
  }
}

// one CTA per position and 256 columns: the first position of a token sums all of its positions, in order
template <bool DROP>
__global__ void __launch_bounds__(256) embedding_bwd_kernel(const float* __restrict__ g, const int32_t* __restrict__ ids,
                                                            int n, int V, int D, float scale, float* __restrict__ dW,
                                                            vtlb_mask m, int accumulate) {
  const int j = blockIdx.x, c = blockIdx.y * 256 + threadIdx.x, id = ids[j];
  if (id < 0 || id >= V) return;
  bool earlier = false;
  for (int k = threadIdx.x; k < j; k += 256) earlier |= ids[k] == id;
  if (__syncthreads_or(earlier) || c >= D) return;
  float sum = 0.0f;
  for (int k = j; k < n; ++k) {
    if (ids[k] != id) continue;
    const size_t e = (size_t)k * D + c;
    float v = g[e];
    if (DROP) {
      const uint4 r = vtlb_philox(m, e / 4);
      v = vtlb_drop(m, e % 4 == 0 ? r.x : e % 4 == 1 ? r.y : e % 4 == 2 ? r.z : r.w, v);
    }
    sum = __fadd_rn(sum, v);
  }
  float* out = dW + (size_t)id * D + c;
  sum = __fmul_rn(sum, scale);
  *out = accumulate ? __fadd_rn(*out, sum) : sum;
}

__global__ void __launch_bounds__(256) ids_from_f32_kernel(const float* __restrict__ src, size_t n, int32_t* __restrict__ ids) {
  for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) {
    const float v = src[i];
    ids[i] = v >= 0.0f && v < 2147483648.0f && v == truncf(v) ? (int32_t)v : -1;
  }
}

int grid_for(vtlb_ctx* ctx, size_t items) {
  const size_t b = (items + 255) / 256, cap = (size_t)ctx->sm_count * 16;
  return (int)(b > cap ? cap : b < 1 ? 1 : b);
}

int check_sizes(vtlb_ctx* ctx, const char* fn, int V, int D, size_t n, double p) {
  if (V <= 0 || D <= 0) return vtlb_fail(ctx, VTLB_EINVAL, "%s: bad table V=%d D=%d", fn, V, D);
  if (n > 0x7fffffffu) return vtlb_fail(ctx, VTLB_EINVAL, "%s: more than 2^31 - 1 positions", fn);
  if (!(p >= 0.0 && p <= 1.0)) return vtlb_fail(ctx, VTLB_EINVAL, "%s: p must be in [0, 1]", fn);
  return VTLB_OK;
}

}  // namespace

VTLB_API int vtlb_embedding_fwd_f32(vtlb_ctx* ctx, const void* d_W, int V, int D, const void* d_ids_i32, size_t n,
                                    float scale, double p, uint64_t seed, uint64_t step, void* d_Y, int check) {
  VTLB_ENTER(ctx);
  if (int rc = check_sizes(ctx, "vtlb_embedding_fwd_f32", V, D, n, p)) return rc;
  if (n == 0) return VTLB_OK;
  if (!d_W || !d_ids_i32 || !d_Y) return vtlb_fail(ctx, VTLB_EINVAL, "vtlb_embedding_fwd_f32: null pointer");
  const size_t total = n * (size_t)D;
  if (vtlb_overlap(d_W, (size_t)V * D, d_Y, total) || vtlb_overlap(d_ids_i32, n, d_Y, total))
    return vtlb_fail(ctx, VTLB_EINVAL, "vtlb_embedding_fwd_f32: the result overlaps an input");
  uint32_t* bad = nullptr;
  vtlb_workspace ws(ctx);
  if (check) {
    bool capturing = false;
    if (int rc = vtlb_capturing(ctx, &capturing)) return rc;
    if (capturing)
      return vtlb_fail(ctx, VTLB_ESTATE, "vtlb_embedding_fwd_f32: check blocks, which a stream under capture cannot");
    void* p_bad = nullptr;
    if (int rc = ws.get(sizeof(uint32_t), &p_bad)) return rc;
    bad = (uint32_t*)p_bad;
    VTLB_CUDA(ctx, cudaMemsetAsync(bad, 0, sizeof(uint32_t), ctx->stream));
  }
  const vtlb_mask m = vtlb_make_mask(p, seed, step);
  auto kern = m.any ? embedding_fwd_kernel<true> : embedding_fwd_kernel<false>;
  kern<<<grid_for(ctx, (total + 3) / 4), 256, 0, ctx->stream>>>((const float*)d_W, V, (uint32_t)D, (const int32_t*)d_ids_i32,
                                                                total, scale, (float*)d_Y, m, bad);
  VTLB_LAUNCHED(ctx);
  if (check) {
    uint32_t flag = 0;
    VTLB_CUDA(ctx, cudaMemcpyAsync(&flag, bad, sizeof flag, cudaMemcpyDeviceToHost, ctx->stream));
    VTLB_CUDA(ctx, cudaStreamSynchronize(ctx->stream));
    if (flag) return vtlb_fail(ctx, VTLB_EINVAL, "vtlb_embedding_fwd_f32: a token is outside [0, %d)", V);
  }
  return VTLB_OK;
}

VTLB_API int vtlb_embedding_bwd_f32(vtlb_ctx* ctx, const void* d_G, const void* d_ids_i32, size_t n, int V, int D,
                                    float scale, double p, uint64_t seed, uint64_t step, void* d_dW, int accumulate) {
  VTLB_ENTER(ctx);
  if (int rc = check_sizes(ctx, "vtlb_embedding_bwd_f32", V, D, n, p)) return rc;
  if (!d_dW || (n && (!d_G || !d_ids_i32))) return vtlb_fail(ctx, VTLB_EINVAL, "vtlb_embedding_bwd_f32: null pointer");
  const size_t table = (size_t)V * D;
  if (vtlb_overlap(d_dW, table, d_G, n * D) || vtlb_overlap(d_dW, table, d_ids_i32, n))
    return vtlb_fail(ctx, VTLB_EINVAL, "vtlb_embedding_bwd_f32: the gradient overlaps an input");
  if (!accumulate) VTLB_CUDA(ctx, cudaMemsetAsync(d_dW, 0, table * sizeof(float), ctx->stream));
  if (n == 0) return VTLB_OK;
  const vtlb_mask m = vtlb_make_mask(p, seed, step);
  auto kern = m.any ? embedding_bwd_kernel<true> : embedding_bwd_kernel<false>;
  kern<<<dim3((unsigned)n, (D + 255) / 256), 256, 0, ctx->stream>>>((const float*)d_G, (const int32_t*)d_ids_i32, (int)n,
                                                                   V, D, scale, (float*)d_dW, m,
                                                                   accumulate);
  VTLB_LAUNCHED(ctx);
  return VTLB_OK;
}

VTLB_API int vtlb_ids_from_f32(vtlb_ctx* ctx, const void* d_src, size_t n, void* d_ids_i32) {
  VTLB_ENTER(ctx);
  if (n == 0) return VTLB_OK;
  if (!d_src || !d_ids_i32) return vtlb_fail(ctx, VTLB_EINVAL, "vtlb_ids_from_f32: null pointer");
  ids_from_f32_kernel<<<grid_for(ctx, n), 256, 0, ctx->stream>>>((const float*)d_src, n, (int32_t*)d_ids_i32);
  VTLB_LAUNCHED(ctx);
  return VTLB_OK;
}
