// Embedding: y[j, :] = scale * W[ids[j], :], with or without dropout on the result (philox.cuh; the mask's element is
// the flat index in y), and its gradient dW[v, :] = scale * sum of the (masked) g[j, :] over the positions j of v.
// A position whose id lies outside the table (padding) gives a row of zeros and takes part in no gradient.
#include <cooperative_groups.h>

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

// ---------------------------------------------------------------- gradient
// The positions are sorted by token (stable: those of a token stay in order), then read in that order, so that a sum is
// a run of consecutive rows and no two threads add to one place: no atomics, the same bits every time.  Three launches:
//   sort   one thread-block cluster; the pairs (token, position) stay in its shared memory over all passes
//   sums   the sorted positions in tiles of equal length whatever the tokens are; a run inside a tile is written to dW,
//          a run that crosses a tile's edge leaves a partial row per tile.  Rows of tokens that do not occur are
//          zeroed by further CTAs of the same launch
//   join   the partial rows of each run that crosses edges, in order
// Bound by HBM: the rows of g that count are read once and dW is written once.
constexpr int kSortThreads = 1024, kSortItemsMax = 16, kSortCtas = 8;
constexpr int kSortMax = kSortThreads * kSortItemsMax * kSortCtas;  // positions per batch; longer calls take several
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;

size_t sort_smem(int items) {
  return (size_t)items * kSortThreads * 8 + (size_t)32 * kDigits * 4 + (size_t)kDigits * 8 + 32 * 4;
}

// Radix sort of (token, position), least significant digit first.  CTA r of the cluster holds elements
// [r, r + 1) * 1024 * ITEMS of the current order, a warp 32 * ITEMS consecutive ones of them.  Tokens outside [0, V)
// take the key V and end up behind all others.  `present`, where given, gets 1 for each token that occurs.
template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads) token_sort_kernel(const int32_t* __restrict__ ids, int n, int V, int passes,
                                                                  int bits, int32_t* __restrict__ sorted_id,
                                                                  int32_t* __restrict__ sorted_pos, uint8_t* present) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  constexpr int kChunk = kSortThreads * ITEMS;
  extern __shared__ uint32_t sm[];
  uint32_t* sm_key = sm;                       // [kChunk]
  uint32_t* sm_pos = sm_key + kChunk;          // [kChunk]
  uint32_t* sm_cnt = sm_pos + kChunk;          // [32 warps][kDigits]
  uint32_t* sm_tot = sm_cnt + 32 * kDigits;    // [kDigits] this CTA's counts
  uint32_t* sm_base = sm_tot + kDigits;        // [kDigits] where this CTA's elements of a digit start
  uint32_t* sm_scan = sm_base + kDigits;       // [32]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int me = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const int first = warp * 32 * ITEMS + lane;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early: the kernel in front is done from here on
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (present) {
    for (size_t i = (size_t)me * kSortThreads + tid; i < ((size_t)V + 15) / 16; i += (size_t)ctas * kSortThreads)
      reinterpret_cast<uint4*>(present)[i] = make_uint4(0, 0, 0, 0);
    __threadfence();
    cluster.sync();
  }
  uint32_t key[ITEMS], pos[ITEMS], rank[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int j = me * kChunk + first + 32 * i;
    const int id = j < n ? ids[j] : -1;
    const bool in = id >= 0 && id < V;
    key[i] = in ? (uint32_t)id : (uint32_t)V;
    pos[i] = (uint32_t)j;
    if (in && present) present[id] = 1;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    const uint32_t mask = (1u << bits) - 1u;
    uint32_t* cnt = sm_cnt + warp * kDigits;
    for (int d = lane; d < kDigits; d += 32) cnt[d] = 0;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint32_t d = (key[i] >> shift) & mask;
      const uint32_t peers = __match_any_sync(0xffffffffu, d);
      const uint32_t before = cnt[d];
      __syncwarp();
      if (lane == __ffs(peers) - 1) cnt[d] = before + __popc(peers);
      rank[i] = before + __popc(peers & ((1u << lane) - 1u));
      __syncwarp();
    }
    __syncthreads();
    uint32_t total = 0;
    if (tid < kDigits) {
      for (int w = 0; w < 32; ++w) {
        const uint32_t c = sm_cnt[w * kDigits + tid];
        sm_cnt[w * kDigits + tid] = total;
        total += c;
      }
      sm_tot[tid] = total;
    }
    cluster.sync();  // the totals of all CTAs are there, and nobody reads its elements from shared memory any more
    uint32_t in_front = 0, all = 0;
    if (tid < kDigits) {
      for (int r = 0; r < ctas; ++r) {
        const uint32_t c = cluster.map_shared_rank(sm_tot, r)[tid];
        if (r < me) in_front += c;
        all += c;
      }
    }
    uint32_t incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sm_scan[warp] = incl;
    __syncthreads();
    if (warp == 0) {
      uint32_t v = sm_scan[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      sm_scan[lane] = v;
    }
    __syncthreads();
    if (tid < kDigits) sm_base[tid] = (warp ? sm_scan[warp - 1] : 0u) + incl - all + in_front;
    __syncthreads();
    const bool out = pass == passes - 1;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint32_t d = (key[i] >> shift) & mask;
      const uint32_t to = sm_base[d] + cnt[d] + rank[i];
      if (out) {
        if (to < (uint32_t)n) sorted_id[to] = (int32_t)key[i], sorted_pos[to] = (int32_t)pos[i];
      } else {
        const int r = (int)(to / kChunk);
        cluster.map_shared_rank(sm_key, r)[to % kChunk] = key[i];
        cluster.map_shared_rank(sm_pos, r)[to % kChunk] = pos[i];
      }
    }
    cluster.sync();  // the elements are in place; and no CTA leaves while another still reads its totals
    if (!out) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) key[i] = sm_key[first + 32 * i], pos[i] = sm_pos[first + 32 * i];
    }
  }
}

struct EmbGrad {
  const float* g;
  const int32_t *sorted_id, *sorted_pos;
  const uint8_t* present;  // null: rows of absent tokens are left alone
  float* dW;
  float* partial;  // [tiles][2][cols * 4]
  size_t first_pos;  // position 0 of this batch in the whole call (the mask's index)
  int n, V, D, cols, tile, tiles;  // cols = ceil(D / 4)
  int slab, slabs, per_cta;        // columns of four per slab, slabs, tiles per CTA
  float scale;
  int accumulate;
};

// Four consecutive values of a row from column 4 * c on; VEC: the rows are 16-byte aligned.
template <bool VEC>
__device__ __forceinline__ float4 row_load(const float* row, int c, int D) {
  if (VEC) return __ldg(reinterpret_cast<const float4*>(row) + c);
  const float* p = row + 4 * c;
  const int left = D - 4 * c;
  return make_float4(__ldg(p), left > 1 ? __ldg(p + 1) : 0.f, left > 2 ? __ldg(p + 2) : 0.f, left > 3 ? __ldg(p + 3) : 0.f);
}
template <bool VEC>
__device__ __forceinline__ void row_store(float* row, int c, int D, float4 v, int accumulate) {
  if (VEC) {
    float4* p = reinterpret_cast<float4*>(row) + c;
    if (accumulate) {
      const float4 o = *p;
      v = make_float4(__fadd_rn(o.x, v.x), __fadd_rn(o.y, v.y), __fadd_rn(o.z, v.z), __fadd_rn(o.w, v.w));
    }
    *p = v;
    return;
  }
  float* p = row + 4 * c;
  const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (4 * c + k < D) p[k] = accumulate ? __fadd_rn(p[k], e[k]) : e[k];
}
// The mask on four consecutive elements from flat index e on (e % 4 = 0 where VEC).
template <bool VEC>
__device__ __forceinline__ float4 drop_at(const vtlb_mask& m, size_t e, float4 v) {
  if (VEC) return vtlb_drop4(m, e / 4, v);
  const uint4 a = vtlb_philox(m, e / 4);
  const int o = (int)(e & 3);
  uint4 w = a;
  if (o) {
    const uint4 b = vtlb_philox(m, e / 4 + 1);
    w = o == 1 ? make_uint4(a.y, a.z, a.w, b.x) : o == 2 ? make_uint4(a.z, a.w, b.x, b.y) : make_uint4(a.w, b.x, b.y, b.z);
  }
  return make_float4(vtlb_drop(m, w.x, v.x), vtlb_drop(m, w.y, v.y), vtlb_drop(m, w.z, v.z), vtlb_drop(m, w.w, v.w));
}
__device__ __forceinline__ void add4(float4& a, float4 v) {
  a = make_float4(__fadd_rn(a.x, v.x), __fadd_rn(a.y, v.y), __fadd_rn(a.z, v.z), __fadd_rn(a.w, v.w));
}
__device__ __forceinline__ float4 mul4(float4 a, float s) {
  return make_float4(__fmul_rn(a.x, s), __fmul_rn(a.y, s), __fmul_rn(a.z, s), __fmul_rn(a.w, s));
}

constexpr int kZeroPerThread = 16;  // columns of four zeroed per thread

template <bool VEC, bool DROP>
__global__ void __launch_bounds__(256) embedding_sums_kernel(EmbGrad p, vtlb_mask m, unsigned sum_ctas) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (blockIdx.x >= sum_ctas) {  // zeros: blocks of four elements of dW, 16-byte aligned where VEC
    const size_t total = (size_t)p.V * p.D;
    const size_t base = (size_t)(blockIdx.x - sum_ctas) * blockDim.x * kZeroPerThread * 4;
    const size_t row0 = base / p.D;
    const uint32_t col0 = (uint32_t)(base - row0 * p.D);
#pragma unroll 4
    for (int i = 0; i < kZeroPerThread; ++i) {
      const uint32_t off = (i * blockDim.x + threadIdx.x) * 4;
      const size_t e = base + off;
      if (e >= total) return;
      if (VEC) {
        if (!p.present[row0 + ((uint64_t)col0 + off) / (uint32_t)p.D]) *reinterpret_cast<float4*>(p.dW + e) = make_float4(0, 0, 0, 0);
      } else {
        for (int k = 0; k < 4 && e + k < total; ++k)
          if (!p.present[row0 + ((uint64_t)col0 + off + k) / (uint32_t)p.D]) p.dW[e + k] = 0.0f;
      }
    }
    return;
  }
  const int group = threadIdx.x / p.slab, c = (int)(blockIdx.x % p.slabs) * p.slab + threadIdx.x % p.slab;
  const int t = (int)(blockIdx.x / p.slabs) * p.per_cta + group;
  if (group >= p.per_cta || t >= p.tiles || c >= p.cols) return;
  const int k0 = t * p.tile, k1 = min(p.n, k0 + p.tile);
  int cur = __ldg(p.sorted_id + k0);
  if (cur >= p.V) return;
  bool starts = k0 == 0 || __ldg(p.sorted_id + k0 - 1) != cur;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int U = 8;
  for (int k = k0; k < k1; k += U) {
    int id[U];
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      id[u] = k + u < k1 ? __ldg(p.sorted_id + k + u) : p.V;
      if (id[u] < p.V) {
        const size_t j = (size_t)__ldg(p.sorted_pos + k + u);
        v[u] = row_load<VEC>(p.g + j * p.D, c, p.D);
        if (DROP) v[u] = drop_at<VEC>(m, (p.first_pos + j) * p.D + 4 * (size_t)c, v[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (id[u] != cur && cur < p.V) {  // the run ends at k + u
        // (at the end of the tile it may go on in the next one)
        const bool ends = k + u < k1 || k1 == p.n || __ldg(p.sorted_id + k1) != cur;
        if (starts && ends)
          row_store<VEC>(p.dW + (size_t)cur * p.D, c, p.D, mul4(acc, p.scale), p.accumulate);
        else
          reinterpret_cast<float4*>(p.partial)[((size_t)t * 2 + starts) * p.cols + c] = acc;
        cur = id[u];
        starts = true;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      if (id[u] < p.V) add4(acc, v[u]);
    }
  }
  if (cur < p.V) {  // a tile whose length is a multiple of U
    const bool ends = k1 == p.n || __ldg(p.sorted_id + k1) != cur;
    if (starts && ends)
      row_store<VEC>(p.dW + (size_t)cur * p.D, c, p.D, mul4(acc, p.scale), p.accumulate);
    else
      reinterpret_cast<float4*>(p.partial)[((size_t)t * 2 + starts) * p.cols + c] = acc;
  }
}

// One CTA per tile and 32 columns of four: where a run starts in tile t and goes on in tile t + 1, its partial rows are
// added up, eight stretches of them at a time, and the stretches in order.
template <bool VEC>
__global__ void __launch_bounds__(256) embedding_join_kernel(EmbGrad p) {
  __shared__ float4 sm[8][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int wide = (p.cols + 31) / 32;
  const int t = (int)(blockIdx.x / wide), k0 = t * p.tile, k1 = k0 + p.tile;
  if (k1 >= p.n) return;
  const int id = __ldg(p.sorted_id + k1 - 1);
  if (id >= p.V || __ldg(p.sorted_id + k1) != id) return;
  if (__ldg(p.sorted_id + k0) == id && k0 > 0 && __ldg(p.sorted_id + k0 - 1) == id) return;  // it started before tile t
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, c = (int)(blockIdx.x % wide) * 32 + lane;
  int more = 1;  // tiles t + 1 .. t + more hold partial rows of it
  for (;;) {
    const size_t k = (size_t)(t + more + 1 + lane) * p.tile;
    const uint32_t differs = __ballot_sync(0xffffffffu, k >= (size_t)p.n || __ldg(p.sorted_id + k) != id);
    if (differs) {
      more += __ffs(differs) - 1;
      break;
    }
    more += 32;
  }
  const float4* rows = reinterpret_cast<const float4*>(p.partial) + (size_t)t * 2 * p.cols + c;
  const int share = (more + 8) / 8;  // of more + 1 rows: the start in slot 1 of tile t, then slot 0 of the others
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < p.cols) {
#pragma unroll 4
    for (int r = part * share; r < min(more + 1, (part + 1) * share); ++r)
      add4(acc, rows[((size_t)r * 2 + (r == 0)) * p.cols]);
  }
  sm[part][lane] = acc;
  __syncthreads();
  if (part || c >= p.cols) return;
  for (int q = 1; q * share <= more; ++q) add4(acc, sm[q][lane]);
  row_store<VEC>(p.dW + (size_t)id * p.D, c, p.D, mul4(acc, p.scale), p.accumulate);
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

template <int ITEMS>
cudaError_t sort_launch(vtlb_ctx* ctx, int ctas, const int32_t* ids, int n, int V, int passes, int bits, int32_t* sorted_id,
                        int32_t* sorted_pos, uint8_t* present) {
  auto kern = token_sort_kernel<ITEMS>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sort_smem(ITEMS));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = sort_smem(ITEMS);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, ids, n, V, passes, bits, sorted_id, sorted_pos, present);
}

int embedding_bwd_batch(vtlb_ctx* ctx, vtlb_workspace& ws, const float* g, const int32_t* ids, size_t first_pos, int n, int V,
                        int D, float scale, const vtlb_mask& m, float* dW, int accumulate) {
  EmbGrad p = {};
  p.g = g, p.dW = dW, p.first_pos = first_pos, p.n = n, p.V = V, p.D = D, p.scale = scale, p.accumulate = accumulate;
  p.cols = (D + 3) / 4;
  p.slabs = (p.cols + 255) / 256;
  p.slab = (p.cols + p.slabs - 1) / p.slabs;
  p.per_cta = 256 / p.slab;
  const int threads = (p.slab * p.per_cta + 31) / 32 * 32;
  p.tile = 32;
  p.tiles = (n + p.tile - 1) / p.tile;
  const size_t list = vtlb_round_up((size_t)n * 4, 256), flags = accumulate ? 0 : vtlb_round_up((size_t)V, 256);
  void* scr = nullptr;
  if (int rc = ws.get(2 * list + flags + (size_t)p.tiles * 2 * p.cols * 16, &scr)) return rc;
  char* at = (char*)scr;
  int32_t *sorted_id = (int32_t*)at, *sorted_pos = (int32_t*)(at + list);
  uint8_t* present = accumulate ? nullptr : (uint8_t*)(at + 2 * list);
  p.sorted_id = sorted_id, p.sorted_pos = sorted_pos, p.present = present;
  p.partial = (float*)(at + 2 * list + flags);

  int key_bits = 1;
  while (key_bits < 31 && (V >> key_bits)) ++key_bits;  // keys 0 .. V
  const int passes = (key_bits + kDigitBits - 1) / kDigitBits, bits = (key_bits + passes - 1) / passes;
  int items = 1;
  while (items * kSortThreads * kSortCtas < n) items *= 2;
  int ctas = 1;
  while (ctas * items * kSortThreads < n) ctas *= 2;
  cudaError_t e;
  switch (items) {
    case 1: e = sort_launch<1>(ctx, ctas, ids, n, V, passes, bits, sorted_id, sorted_pos, present); break;
    case 2: e = sort_launch<2>(ctx, ctas, ids, n, V, passes, bits, sorted_id, sorted_pos, present); break;
    case 4: e = sort_launch<4>(ctx, ctas, ids, n, V, passes, bits, sorted_id, sorted_pos, present); break;
    case 8: e = sort_launch<8>(ctx, ctas, ids, n, V, passes, bits, sorted_id, sorted_pos, present); break;
    default: e = sort_launch<16>(ctx, ctas, ids, n, V, passes, bits, sorted_id, sorted_pos, present); break;
  }
  VTLB_CUDA(ctx, e);
  VTLB_LAUNCHED(ctx);

  const bool vec = D % 4 == 0 && vtlb_aligned16(g) && vtlb_aligned16(dW);
  const unsigned sum_ctas = (unsigned)((p.tiles + p.per_cta - 1) / p.per_cta) * p.slabs;
  const size_t per_zero = (size_t)threads * kZeroPerThread * 4, table = (size_t)V * D;
  const size_t zero_ctas = accumulate ? 0 : (table + per_zero - 1) / per_zero;
  auto sums = vec ? (m.any ? embedding_sums_kernel<true, true> : embedding_sums_kernel<true, false>)
                  : (m.any ? embedding_sums_kernel<false, true> : embedding_sums_kernel<false, false>);
  VTLB_CUDA(ctx, vtlb_launch_early(sums, dim3((unsigned)(sum_ctas + zero_ctas)), dim3(threads), 0, ctx->stream, p, m, sum_ctas));
  VTLB_LAUNCHED(ctx);
  if (p.tiles > 1) {
    auto join = vec ? embedding_join_kernel<true> : embedding_join_kernel<false>;
    VTLB_CUDA(ctx, vtlb_launch_early(join, dim3((unsigned)(p.tiles - 1) * ((p.cols + 31) / 32)), dim3(256), 0, ctx->stream, p));
    VTLB_LAUNCHED(ctx);
  }
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
  if (n == 0) {
    if (!accumulate) VTLB_CUDA(ctx, cudaMemsetAsync(d_dW, 0, table * sizeof(float), ctx->stream));
    return VTLB_OK;
  }
  vtlb_workspace ws(ctx);
  const vtlb_mask m = vtlb_make_mask(p, seed, step);
  for (size_t at = 0; at < n; at += kSortMax) {
    const int count = (int)(n - at < kSortMax ? n - at : kSortMax);
    if (int rc = embedding_bwd_batch(ctx, ws, (const float*)d_G + at * D, (const int32_t*)d_ids_i32 + at, at, count, V, D,
                                     scale, m, (float*)d_dW, accumulate || at))
      return rc;
  }
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
