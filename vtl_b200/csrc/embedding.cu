// Embedding: y[j, :] = scale * W[ids[j], :], with or without dropout on the result (philox.cuh; the mask's element is
// the flat index in y), and its gradient dW[v, :] = scale * sum of the (masked) g[j, :] over the positions j of v.
// A position whose id lies outside the table (padding) gives a row of zeros and takes part in no gradient.
#include <cooperative_groups.h>

#include "philox.cuh"

namespace {

// Four consecutive elements of y per step, U steps at a time: bound by HBM (a row of W in, a row of y out), so what counts is
// that every thread has U loads in flight.  VEC: D is a multiple of four and both arrays are 16-byte aligned, so that
// the four lie in one row.  16384 rows of 4096 out of 50000: 63 us, 5.9 TB/s, 90 % of a plain copy's rate (a simple
// kernel with one load in flight: 170 us).  999 rows of 2047 with dropout: 6.2 us, of which the mask's ten dependent rounds and
// the loads of ids and rows behind one another leave little to gain.  Eight rows of 4096: 4.5 us, the host's call.
template <bool VEC, bool DROP, int U>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(const float* __restrict__ W, int V, uint32_t D,
                                                            const int32_t* __restrict__ ids, size_t total, float scale,
                                                            float* __restrict__ y, bool blocks_of_w, bool y_aligned, vtlb_mask m,
                                                            uint32_t* bad) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early: the kernel in front is done from here on
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const size_t first = (size_t)blockIdx.x * (256 * 4 * U);  // element of y
  const size_t row0 = first / D;
  const uint32_t col0 = (uint32_t)(first - row0 * D);  // D + 4096 * U fits 32 bits: D < 2^31
  float v[U][4];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t off = col0 + (u * 256 + threadIdx.x) * 4;
    uint32_t row = off / D, col = off - row * D;
    size_t j = row0 + row;
    if (first + (size_t)(u * 256 + threadIdx.x) * 4 >= total) {
      v[u][0] = v[u][1] = v[u][2] = v[u][3] = 0.0f;
      continue;
    }
    int id = __ldg(ids + j);
    bool in = id >= 0 && id < V;
    if (!in && bad) atomicOr(bad, 1u);
    if (VEC) {
      const float4 f = in ? __ldg(reinterpret_cast<const float4*>(W + (size_t)id * D + col)) : make_float4(0, 0, 0, 0);
      v[u][0] = f.x, v[u][1] = f.y, v[u][2] = f.z, v[u][3] = f.w;
    } else if (blocks_of_w && in && col + 4 <= D && ((size_t)id * D + col) / 4 * 4 + 8 <= (size_t)V * D) {
      // all of one row: the two aligned blocks that hold them (a neighbour's, too, so that HBM sees each once)
      const size_t at = (size_t)id * D + col;
      const uint32_t o = (uint32_t)at & 3;
      const float4* blocks = reinterpret_cast<const float4*>(W) + at / 4;
      const float4 a = __ldg(blocks), b = o ? __ldg(blocks + 1) : a;
      v[u][0] = o == 0 ? a.x : o == 1 ? a.y : o == 2 ? a.z : a.w;
      v[u][1] = o == 0 ? a.y : o == 1 ? a.z : o == 2 ? a.w : b.x;
      v[u][2] = o == 0 ? a.z : o == 1 ? a.w : o == 2 ? b.x : b.y;
      v[u][3] = o == 0 ? a.w : o == 1 ? b.x : o == 2 ? b.y : b.z;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[u][k] = in && j * D + col < total ? __ldg(W + (size_t)id * D + col) : 0.0f;
        if (++col == D && j * D + col < total) {  // the next row
          col = 0;
          id = __ldg(ids + ++j);
          in = id >= 0 && id < V;
          if (!in && bad) atomicOr(bad, 1u);
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const size_t e = first + (size_t)(u * 256 + threadIdx.x) * 4;
    if (e >= total) return;
    float4 o = make_float4(__fmul_rn(v[u][0], scale), __fmul_rn(v[u][1], scale), __fmul_rn(v[u][2], scale),
                           __fmul_rn(v[u][3], scale));
    if (DROP) o = vtlb_drop4(m, e / 4, o);
    if (VEC || (y_aligned && e + 4 <= total)) {
      *reinterpret_cast<float4*>(y + e) = o;
    } else {
      const float q[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e + k < total) y[e + k] = q[k];
    }
  }
}

// ---------------------------------------------------------------- gradient
// The positions are sorted by token (stable: those of a token stay in order), then read in that order, so that a sum is
// a run of consecutive rows and no two threads add to one place: no atomics, the same bits every time.  Three launches, or
// one where there are few positions (embedding_few_kernel):
//   sort   pairs (token, position); tokens outside [0, V) take the key V and end up behind all others
//   sums   the sorted positions in tiles of equal length whatever the tokens are.  A run that ends within a tile's
//          length of the tile it starts in is summed there as a whole; a longer one leaves a partial row per tile.
//          Rows of tokens that do not occur are zeroed by further CTAs of this launch, which need nothing of the sort and
//          start while it runs
//   join   the partial rows of each long run, in order
// Bound by HBM: the rows of g that count are read once and dW is written once.  16384 x 4096 into 50000 rows: 186 us,
// 5.8 TB/s, 89 % of a plain copy's rate.  8191 x 1023 with a mask into 3001 rows: 41 us against 5.7 of bytes; there it is
// the sort (10 us, partly beside the zeroing), two rounds of loads and masks per tile with 20 warps on an SM (some 25), and
// the join (7) behind one another.

// Sort of up to kRankMax positions: a warp finds the ranks of four of them by comparing with all.  n^2 comparisons, two
// instructions each, spread over the whole GPU, against two or three passes of a few microseconds each on one cluster.
// (2000 positions x 1023: 20.6 us in all, 22.8 by way of the cluster; 4000: 32.5 and 31.3.)
constexpr int kRankMax = 2048;
__global__ void __launch_bounds__(256) token_rank_kernel(const int32_t* __restrict__ ids, int n, int V, int2* __restrict__ sorted) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, j0 = (int)(blockIdx.x * 8 + (threadIdx.x >> 5)) * 4;
  if (j0 >= n) return;
  const auto key_at = [&](int i) {
    const int id = i < n ? __ldg(ids + i) : -1;
    return id >= 0 && id < V ? (uint32_t)id : (uint32_t)V;
  };
  uint32_t key[4];
  int rank[4] = {0, 0, 0, 0};
#pragma unroll
  for (int q = 0; q < 4; ++q) key[q] = key_at(j0 + q);
  const int own = j0 & ~31;  // the 32 positions around j0 .. j0 + 3
#pragma unroll 4
  for (int i = lane; i < own; i += 32) {
    const uint32_t k = key_at(i);
#pragma unroll
    for (int q = 0; q < 4; ++q) rank[q] += k <= key[q];
  }
  {
    const int i = own + lane;
    const uint32_t k = key_at(i);
#pragma unroll
    for (int q = 0; q < 4; ++q) rank[q] += i < n && (k < key[q] || (k == key[q] && i < j0 + q));
  }
#pragma unroll 4
  for (int i = own + 32 + lane; i < n; i += 32) {
    const uint32_t k = key_at(i);
#pragma unroll
    for (int q = 0; q < 4; ++q) rank[q] += k < key[q];
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = __reduce_add_sync(0xffffffffu, rank[q]);
    if (lane == q && j0 + q < n) sorted[r] = make_int2((int)key[q], j0 + q);
  }
}

constexpr int kSortThreads = 1024, kSortItemsMax = 16, kSortCtas = 8;
constexpr int kSortMax = kSortThreads * kSortItemsMax * kSortCtas;  // positions per batch; longer calls take several
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;

size_t sort_smem(int items) {
  return (size_t)items * kSortThreads * 8 + (size_t)32 * kDigits * 4 + (size_t)kDigits * 8 + 32 * 4;
}

// Radix sort of more positions, least significant digit first, in the shared memory of one thread-block cluster: CTA r
// holds elements [r, r + 1) * 1024 * ITEMS of the current order, a warp 32 * ITEMS consecutive ones of them.  A pass ranks
// a warp's elements by matching digits, adds up the warps' and CTAs' counts and sends each element to its place in some
// CTA's shared memory; the keys have as many passes of up to nine bits as V needs.  Bound by the latency of the barriers
// in the cluster: 16 us for 16384 positions of 16 bits, during which the zeroing writes 100 MB.
template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads) token_sort_kernel(const int32_t* __restrict__ ids, int n, int V, int passes,
                                                                  int bits, int2* __restrict__ sorted) {
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
  const int first = warp * 32 * ITEMS + lane, digits = 1 << bits;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early: the kernel in front is done from here on
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  uint32_t key[ITEMS], pos[ITEMS], rank[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int j = me * kChunk + first + 32 * i;
    const int id = j < n ? __ldg(ids + j) : -1;
    key[i] = id >= 0 && id < V ? (uint32_t)id : (uint32_t)V;
    pos[i] = (uint32_t)j;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    const uint32_t mask = (uint32_t)digits - 1u;
    uint32_t* cnt = sm_cnt + warp * kDigits;
    for (int d = lane; d < digits; d += 32) cnt[d] = 0;
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
    if (tid < digits) {
      uint32_t c[32], total = 0;
#pragma unroll
      for (int w = 0; w < 32; ++w) c[w] = sm_cnt[w * kDigits + tid];
#pragma unroll
      for (int w = 0; w < 32; ++w) {
        sm_cnt[w * kDigits + tid] = total;
        total += c[w];
      }
      sm_tot[tid] = total;
    }
    cluster.sync();  // the totals of all CTAs are there, and nobody reads its elements from shared memory any more
    uint32_t in_front = 0, all = 0;
    if (tid < digits) {
#pragma unroll
      for (int r = 0; r < kSortCtas; ++r) {
        const uint32_t c = r < ctas ? cluster.map_shared_rank(sm_tot, r)[tid] : 0u;
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
    uint32_t base = 0;  // of the digits of earlier warps; at most kDigits / 32 hold any
#pragma unroll
    for (int w = 0; w < kDigits / 32; ++w) base += w < warp ? sm_scan[w] : 0u;
    if (tid < digits) sm_base[tid] = base + incl - all + in_front;
    __syncthreads();
    const bool out = pass == passes - 1;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint32_t d = (key[i] >> shift) & mask;
      const uint32_t to = sm_base[d] + cnt[d] + rank[i];
      if (out) {
        if (to < (uint32_t)n) sorted[to] = make_int2((int)key[i], (int)pos[i]);
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
  const int32_t* ids;
  const int2* sorted;  // (token, position)
  float* dW;
  float* partial;  // [tiles][2][cols * 4]
  size_t first_pos;  // position 0 of this batch in the whole call (the mask's index)
  int n, V, D, cols, tile, tiles;  // cols = ceil(D / 4)
  int slab, slabs, per_cta;        // columns of four (else: warps) per slab, slabs, tiles per CTA
  float scale;
  int accumulate;
};

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
// Rows that are not 16-byte aligned (D % 4 = o > 0 from one row to the next, or a displaced g): a lane takes the aligned
// block of four elements of g that starts `o` columns before column 4 * c, draws one block of the mask for it, and hands
// its first o elements to the lane before it.  (Four single loads and two blocks of the mask otherwise.)  The last lane
// of a warp only helps the one before it.
__device__ __forceinline__ float4 block_load(const float* g, size_t e, size_t total, bool aligned) {
  if (aligned && e + 4 <= total) return __ldg(reinterpret_cast<const float4*>(g + e));
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (e < total) v.x = __ldg(g + e);
  if (e + 1 < total) v.y = __ldg(g + e + 1);
  if (e + 2 < total) v.z = __ldg(g + e + 2);
  if (e + 3 < total) v.w = __ldg(g + e + 3);
  return v;
}
__device__ __forceinline__ float4 shift_down(float4 v, int o) {  // o is the same in all lanes
  if (o == 0) return v;
  const float x = __shfl_down_sync(0xffffffffu, v.x, 1);
  if (o == 1) return make_float4(v.y, v.z, v.w, x);
  const float y = __shfl_down_sync(0xffffffffu, v.y, 1);
  if (o == 2) return make_float4(v.z, v.w, x, y);
  const float z = __shfl_down_sync(0xffffffffu, v.z, 1);
  return make_float4(v.w, x, y, z);
}
__device__ __forceinline__ void add4(float4& a, float4 v) {
  a = make_float4(__fadd_rn(a.x, v.x), __fadd_rn(a.y, v.y), __fadd_rn(a.z, v.z), __fadd_rn(a.w, v.w));
}
__device__ __forceinline__ float4 mul4(float4 a, float s) {
  return make_float4(__fmul_rn(a.x, s), __fmul_rn(a.y, s), __fmul_rn(a.z, s), __fmul_rn(a.w, s));
}

// Zeros in the rows [row0, row1) of dW whose token does not occur, kZeroRows of them at a time: which do occur is seen from
// all of the ids, by every CTA for itself.
constexpr int kZeroRows = 8192;
__device__ __forceinline__ void zero_absent(const EmbGrad& p, size_t row0, size_t row1) {
  __shared__ uint32_t met[kZeroRows / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (size_t r0 = row0; r0 < row1; r0 += kZeroRows) {
    const int rows = (int)(row1 - r0 < kZeroRows ? row1 - r0 : kZeroRows);
    for (int i = threadIdx.x; i < (rows + 31) / 32; i += blockDim.x) met[i] = 0;
    __syncthreads();
    const auto mark = [&](int id) {
      const int64_t r = (int64_t)id - (int64_t)r0;
      if (r >= 0 && r < rows && !(met[r >> 5] >> (r & 31) & 1u)) atomicOr(&met[r >> 5], 1u << (r & 31));
    };
    // 16-byte pieces of the ids, several in flight: this is latency, during which nothing is written
    const int lead = min(p.n, (int)((16 - ((uintptr_t)p.ids & 15)) & 15) / 4), quads = (p.n - lead) / 4;
    const int4* ids4 = reinterpret_cast<const int4*>(p.ids + lead);
#pragma unroll 8
    for (int i = threadIdx.x; i < quads; i += blockDim.x) {
      const int4 q = __ldg(ids4 + i);
      mark(q.x), mark(q.y), mark(q.z), mark(q.w);
    }
    if ((int)threadIdx.x < lead) mark(__ldg(p.ids + threadIdx.x));
    if ((int)threadIdx.x < p.n - lead - 4 * quads) mark(__ldg(p.ids + lead + 4 * quads + threadIdx.x));
    __syncthreads();
    if (p.cols >= 32) {  // a warp per row, 16 bytes per lane but for the row's unaligned ends
      for (int r = warp; r < rows; r += blockDim.x >> 5) {
        if (met[r >> 5] >> (r & 31) & 1u) continue;
        float* row = p.dW + (r0 + r) * p.D;
        const int head = (int)((16 - ((uintptr_t)row & 15)) & 15) / 4, body = (p.D - head) / 4, end = head + 4 * body;
        float4* out = reinterpret_cast<float4*>(row + head);
#pragma unroll 4
        for (int c = lane; c < body; c += 32) out[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (lane < head) row[lane] = 0.0f;
        if (lane < p.D - end) row[end + lane] = 0.0f;
      }
    } else {  // element by element, a warp's 32 next to one another
      float* out = p.dW + r0 * p.D;
      const uint32_t D = (uint32_t)p.D, total = (uint32_t)rows * D, dr = blockDim.x / D, dc = blockDim.x - dr * D;
      uint32_t r = threadIdx.x / D, c = threadIdx.x - r * D;
      for (uint32_t e = threadIdx.x; e < total; e += blockDim.x) {
        if (!(met[r >> 5] >> (r & 31) & 1u)) out[e] = 0.0f;
        r += dr, c += dc;
        if (c >= D) c -= D, ++r;
      }
    }
    __syncthreads();
  }
}

// Few positions in one launch, without a sort: a warp finds the positions of the token of position j by comparing with all,
// and where j is the first of them it sums 128 columns of their rows (eight rows at a time, in order).  More than kFewAlone
// rows are summed by all warps of the CTA, an eighth each.  Rows of absent tokens are zeroed by further CTAs.  Bound by
// latency: the host's launch, the ids, a row of g.
// 256 positions x 600, 5000 tokens: 5.1 us, 10.4 by way of the sort; 1024 x 600: 9.0 and 13.0; 512 x 4096: 23.0 and 27.8;
// 2048 x 512: 30.0 and 27.1, all of them one token 18.6 and 28.1; 2048 x 1023: 36 and 22 (each CTA compares the positions
// for itself, so many CTAs do so many times).  With a mask, whose blocks leave room for four rows at a time, half as many:
// 2048 x 255: 16.8 and 18.2; 1024 x 1023: 21.1 and 17.9.
constexpr int kFewAlways = 512, kFewMax = 2048, kFewElements = 1 << 20, kFewAlone = 16;
template <bool VEC, bool DROP>
__global__ void __launch_bounds__(256, 4) embedding_few_kernel(EmbGrad p, vtlb_mask m, unsigned zero_ctas) {
  __shared__ int ids[kFewMax];
  __shared__ uint16_t list[8][kFewMax];  // the positions of each warp's token
  __shared__ int count[8];
  __shared__ float4 part[8][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (blockIdx.x < zero_ctas) {
    const size_t each = ((size_t)p.V + zero_ctas - 1) / zero_ctas, row0 = blockIdx.x * each;
    zero_absent(p, row0, row0 + each < (size_t)p.V ? row0 + each : (size_t)p.V);
    return;
  }
  const unsigned cta = blockIdx.x - zero_ctas;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, words = (p.n + 31) / 32;
  // (positions far from one another: tokens met often have their first positions together, at the start)
  const int apart = (p.n + 7) / 8, j0 = (int)(cta / p.slabs), j = j0 + warp * apart;
  const size_t total = (size_t)p.n * p.D;
  const bool aligned = ((uintptr_t)p.g & 15) == 0;
  for (int i = threadIdx.x; i < words * 32; i += 256) {
    const int id = i < p.n ? __ldg(p.ids + i) : -1;
    ids[i] = id < p.V ? id : -1;
  }
  __syncthreads();
  const int id = j < p.n ? ids[j] : -1;
  if (id >= 0) {
    bool first = true;
    for (int i = lane; i < (j & ~31); i += 32) first = first && ids[i] != id;
    first = __all_sync(0xffffffffu, first && ((j & ~31) + lane >= j || ids[(j & ~31) + lane] != id));
    int found = 0;
    if (first)
      for (int i = j / 32; i < words; ++i) {
        const bool hit = ids[i * 32 + lane] == id;
        const uint32_t hits = __ballot_sync(0xffffffffu, hit);
        if (hit) list[warp][found + __popc(hits & ((1u << lane) - 1u))] = (uint16_t)(i * 32 + lane);
        found += __popc(hits);
      }
    if (lane == 0) count[warp] = found;
  } else if (lane == 0) {
    count[warp] = 0;
  }
  __syncwarp();
  const auto sum = [&](const uint16_t* rows, int k0, int k1, int c, bool own) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int U = DROP ? 4 : 8;
    for (int k = k0; k < k1; k += U) {
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k + u < k1) {
          const size_t row = (size_t)rows[k + u] * p.D;
          if (VEC) {
            if (own) v[u] = __ldg(reinterpret_cast<const float4*>(p.g + row) + c);
          } else if (4u * (uint32_t)c < (uint32_t)p.D + (uint32_t)(row & 3)) {
            v[u] = block_load(p.g, (row & ~(size_t)3) + 4 * (size_t)c, total, aligned);
          }
        }
      }
      if (DROP || !VEC) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const size_t e = (p.first_pos + rows[min(k + u, k1 - 1)]) * (size_t)p.D;
          if (DROP) v[u] = vtlb_drop4(m, e / 4 + c, v[u]);
          if (!VEC) v[u] = shift_down(v[u], (int)(e & 3));
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k + u < k1) add4(acc, v[u]);
    }
    return acc;
  };
  constexpr int kWide = VEC ? 32 : 31;
  const int c0 = (int)(cta % p.slabs) * p.slab * kWide, c1 = min(p.cols, c0 + p.slab * kWide);
  const int rows = count[warp];
  if (rows && rows <= kFewAlone)
    for (int c = c0 + lane; c - lane < c1; c += kWide) {
      const bool own = c < p.cols && lane < kWide;
      const float4 acc = sum(list[warp], 0, rows, c, own);
      if (own) row_store<VEC>(p.dW + (size_t)id * p.D, c, p.D, mul4(acc, p.scale), p.accumulate);
    }
  __syncthreads();
  for (int w = 0; w < 8; ++w) {
    const int all = count[w], share = (all + 7) / 8;
    if (all <= kFewAlone) continue;
    for (int c = c0 + lane; c - lane < c1; c += kWide) {
      const bool own = c < p.cols && lane < kWide;
      part[warp][lane] = sum(list[w], warp * share, min(all, (warp + 1) * share), c, own);
      __syncthreads();
      if (warp == 0 && own) {
        float4 acc = part[0][lane];
        for (int q = 1; q * share < all; ++q) add4(acc, part[q][lane]);
        row_store<VEC>(p.dW + (size_t)ids[j0 + w * apart] * p.D, c, p.D, mul4(acc, p.scale), p.accumulate);
      }
      __syncthreads();
    }
  }
}

constexpr int kTileMax = 64, kCtaPositions = 1024;  // positions per tile and per CTA
// (Four CTAs per SM without a mask: 16384 x 4096 186 us in all, 189 with three; with one three: 251 and 255.)
template <bool VEC, bool DROP>
__global__ void __launch_bounds__(256, DROP ? 3 : 4) embedding_sums_kernel(EmbGrad p, vtlb_mask m, unsigned zero_ctas) {
  __shared__ int2 window[kCtaPositions + 2 * kTileMax + 2];  // the sorted positions of this CTA's tiles and a tile around them
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (blockIdx.x < zero_ctas) {
    // No wait for the sort: nothing of it is read here, and it started only when everything in front of it was done.
    const size_t each = ((size_t)p.V + zero_ctas - 1) / zero_ctas, row0 = blockIdx.x * each;
    zero_absent(p, row0, row0 + each < (size_t)p.V ? row0 + each : (size_t)p.V);
    return;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const unsigned cta = blockIdx.x - zero_ctas;
  const int T = p.tile, t0 = (int)(cta / p.slabs) * p.per_cta, w0 = (t0 - 1) * T - 1;
  for (int i = threadIdx.x; i < (p.per_cta + 2) * T + 2; i += blockDim.x)
    window[i] = w0 + i >= 0 && w0 + i < p.n ? __ldg(p.sorted + w0 + i) : make_int2(-1, 0);
  __syncthreads();
  const int unit = VEC ? threadIdx.x : threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = unit / p.slab, at = (int)(cta % p.slabs) * p.slab + unit % p.slab;
  const int c = VEC ? at : at * 31 + lane;
  const int t = t0 + group;
  if (group >= p.per_cta || t >= p.tiles || (VEC ? c : at * 31) >= p.cols) return;  // (whole warps where they shuffle)
  const bool own = VEC || (lane < 31 && c < p.cols);
  const size_t total = (size_t)p.n * p.D;
  const bool aligned = ((uintptr_t)p.g & 15) == 0;
  const int k0 = t * T, k1 = min(p.n, k0 + T);
  const auto id_at = [&](int k) { return window[k - w0].x; };  // -1 before the first and behind the last position
  int cur = id_at(k0);
  if (cur >= p.V) return;
  // The run that comes in from an earlier tile: long if it started before the last tile or goes on into the next one.
  const bool comes_in = id_at(k0 - 1) == cur;
  const bool lead = comes_in && (id_at(k0 - T - 1) == cur || id_at(k0 + T) == cur);
  const int skip = comes_in && !lead ? cur : -1;  // its first tile sums it
  // The run that starts here and goes on into the next tile: short if it ends in that one.
  const int last = id_at(k1 - 1);
  const bool goes_on = last < p.V && id_at(k1) == last && !(comes_in && last == cur);
  const bool tail = goes_on && id_at(k1 + T) == last;
  const int end = goes_on && !tail ? min(p.n, k1 + T) : k1;
  bool first = lead;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const auto flush = [&] {
    if (!own) {
    } else if (first) {
      reinterpret_cast<float4*>(p.partial)[(size_t)t * 2 * p.cols + c] = acc;
    } else if (tail && cur == last) {
      reinterpret_cast<float4*>(p.partial)[((size_t)t * 2 + 1) * p.cols + c] = acc;
    } else if (cur != skip) {
      row_store<VEC>(p.dW + (size_t)cur * p.D, c, p.D, mul4(acc, p.scale), p.accumulate);
    }
    first = false;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
  };
  // token of sorted position k of this tile (V: none)
  const auto token = [&](int k) {
    const int id = k < end ? window[k - w0].x : p.V;
    return k < k1 || id == last ? id : p.V;
  };
  constexpr int U = DROP ? 4 : 8;  // (the mask's block takes the registers of four more rows)
  for (int k = k0; k < end; k += U) {
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int id = token(k + u);
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (id < p.V && id != skip) {
        const size_t row = (size_t)window[k + u - w0].y * p.D;
        if (VEC)
          v[u] = __ldg(reinterpret_cast<const float4*>(p.g + row) + c);
        else if (4u * (uint32_t)c < (uint32_t)p.D + (uint32_t)(row & 3))
          v[u] = block_load(p.g, (row & ~(size_t)3) + 4 * (size_t)c, total, aligned);
      }
    }
    // (all U rows, valid or not, without a branch between them: a block of the mask is a chain of some 150 cycles)
    if (DROP || !VEC) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const size_t e = (p.first_pos + (size_t)window[min(k + u, end - 1) - w0].y) * p.D;
        if (DROP) v[u] = vtlb_drop4(m, e / 4 + c, v[u]);
        if (!VEC) v[u] = shift_down(v[u], (int)(e & 3));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int id = token(k + u);
      if (id != cur) {
        if (cur < p.V) flush();
        cur = id;
      }
      if (id < p.V && id != skip) add4(acc, v[u]);
    }
  }
  if (cur < p.V) flush();
}

// Where a long run starts in tile t, its partial rows (slot 1 of tile t, slot 0 of the following ones) are added up: eight
// stretches of them at a time, and the stretches in order.  A CTA looks after eight tiles (most start no long run, and
// a CTA per tile costs more than the sums) and one of `split` shares of the columns.  Bound by the latency of its few
// loads behind one another: 7 us behind 8191 x 1023.
constexpr int kJoinTiles = 8;
template <bool VEC>
__global__ void __launch_bounds__(256) embedding_join_kernel(EmbGrad p, int split) {
  __shared__ float4 sm[8][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int T = p.tile, t0 = (int)(blockIdx.x / split) * kJoinTiles;
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const auto id_at = [&](long long k) { return k >= 0 && k < p.n ? __ldg(&p.sorted[k].x) : -1; };
  const int own = t0 + (lane & (kJoinTiles - 1));  // every warp sees the starts of all eight tiles
  const int own_id = own < p.tiles ? id_at((long long)own * T + T - 1) : -1;
  const bool starts = own_id >= 0 && own_id < p.V && id_at((long long)own * T + 2 * T) == own_id &&
                      id_at((long long)own * T - 1) != own_id;
  uint32_t todo = __ballot_sync(0xffffffffu, starts) & ((1u << kJoinTiles) - 1u);
  for (; todo; todo &= todo - 1) {
    const int t = t0 + __ffs(todo) - 1, id = __shfl_sync(0xffffffffu, own_id, t - t0);
    int more = 2;  // tiles t + 1 .. t + more hold partial rows of it
    for (;;) {
      const uint32_t differs = __ballot_sync(0xffffffffu, id_at((long long)(t + more + 1 + lane) * T) != id);
      if (differs) {
        more += __ffs(differs) - 1;
        break;
      }
      more += 32;
    }
    const int share = (more + 8) / 8;  // of more + 1 rows
    for (int c0 = (int)(blockIdx.x % split) * 32; c0 < p.cols; c0 += split * 32) {
      const int c = c0 + lane;
      const float4* rows = reinterpret_cast<const float4*>(p.partial) + (size_t)t * 2 * p.cols + c;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c < p.cols) {
#pragma unroll 4
        for (int r = part * share; r < min(more + 1, (part + 1) * share); ++r)
          add4(acc, rows[((size_t)r * 2 + (r == 0)) * p.cols]);
      }
      __syncthreads();
      sm[part][lane] = acc;
      __syncthreads();
      if (part == 0 && c < p.cols) {
        for (int q = 1; q * share <= more; ++q) add4(acc, sm[q][lane]);
        row_store<VEC>(p.dW + (size_t)id * p.D, c, p.D, mul4(acc, p.scale), p.accumulate);
      }
    }
  }
}

__global__ void __launch_bounds__(256) ids_from_f32_kernel(const float* src, size_t n, int32_t* ids) {
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
cudaError_t sort_launch(vtlb_ctx* ctx, int ctas, const int32_t* ids, int n, int V, int passes, int bits, int2* sorted) {
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
  cfg.numAttrs = vtlb_early_on() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, ids, n, V, passes, bits, sorted);
}

cudaError_t sort_positions(vtlb_ctx* ctx, const int32_t* ids, int n, int V, int2* sorted) {
  if (n <= kRankMax) return vtlb_launch_early(token_rank_kernel, dim3((n + 31) / 32), dim3(256), 0, ctx->stream, ids, n, V, sorted);
  int key_bits = 1;
  while (key_bits < 31 && (V >> key_bits)) ++key_bits;  // keys 0 .. V
  const int passes = (key_bits + kDigitBits - 1) / kDigitBits, bits = (key_bits + passes - 1) / passes;
  int items = 1, ctas = 1;
  while (items * kSortThreads * kSortCtas < n) items *= 2;
  while (ctas * items * kSortThreads < n) ctas *= 2;
  switch (items) {
    case 1: return sort_launch<1>(ctx, ctas, ids, n, V, passes, bits, sorted);
    case 2: return sort_launch<2>(ctx, ctas, ids, n, V, passes, bits, sorted);
    case 4: return sort_launch<4>(ctx, ctas, ids, n, V, passes, bits, sorted);
    case 8: return sort_launch<8>(ctx, ctas, ids, n, V, passes, bits, sorted);
    default: return sort_launch<16>(ctx, ctas, ids, n, V, passes, bits, sorted);
  }
}

int embedding_bwd_batch(vtlb_ctx* ctx, vtlb_workspace& ws, const float* g, const int32_t* ids, size_t first_pos, int n, int V,
                        int D, float scale, const vtlb_mask& m, float* dW, int accumulate) {
  EmbGrad p = {};
  p.g = g, p.ids = ids, p.dW = dW, p.first_pos = first_pos, p.n = n, p.V = V, p.D = D, p.scale = scale, p.accumulate = accumulate;
  p.cols = D / 4 + (D % 4 != 0);
  const bool vec = D % 4 == 0 && vtlb_aligned16(g) && vtlb_aligned16(dW);
  // Each zeroing CTA reads all ids, so they are no more than write four times what all of them read, but two per SM
  // where there are 32 KB to write for each.
  const size_t table = (size_t)V * D * 4;
  size_t want = table / ((size_t)n * 16), least = (size_t)2 * ctx->sm_count;
  want = want < least ? least : want;
  if (want > table / 32768 + 1) want = table / 32768 + 1;
  const unsigned zero_ctas = accumulate ? 0u : (unsigned)(want < (size_t)V ? want : (size_t)V);
  if (n <= kFewAlways >> m.any || (n <= kFewMax && (long long)n * D <= kFewElements >> m.any)) {
    // Pieces of 128 columns to a CTA: as many as leave eight CTAs per SM, for each finds its positions for itself.
    const int pieces = vec ? (p.cols + 31) / 32 : (p.cols + 30) / 31;
    p.slab = 1;
    while (p.slab < pieces && (long long)((n + 7) / 8) * pieces > (long long)p.slab * 8 * ctx->sm_count) p.slab *= 2;
    p.slabs = (pieces + p.slab - 1) / p.slab;
    auto few = vec ? (m.any ? embedding_few_kernel<true, true> : embedding_few_kernel<true, false>)
                   : (m.any ? embedding_few_kernel<false, true> : embedding_few_kernel<false, false>);
    VTLB_CUDA(ctx, vtlb_launch_early(few, dim3((unsigned)((n + 7) / 8) * p.slabs + zero_ctas), dim3(256), 0, ctx->stream, p, m, zero_ctas));
    VTLB_LAUNCHED(ctx);
    return VTLB_OK;
  }
  const int units = vec ? p.cols : (p.cols + 30) / 31, most = vec ? 256 : 8;  // threads, or warps, per row and per CTA
  p.slabs = (units + most - 1) / most;
  p.slab = (units + p.slabs - 1) / p.slabs;
  p.per_cta = most / p.slab;
  const int threads = vec ? (p.slab * p.per_cta + 31) / 32 * 32 : p.slab * p.per_cta * 32;
  // Tiles of 4 to 64 positions: long enough that few runs are cut, short enough for eight to sixteen CTAs per SM.
  p.tile = 4;
  while (p.tile < kTileMax && p.tile * 2 * p.per_cta <= kCtaPositions && (long long)n * p.slabs > (long long)p.tile * p.per_cta * 16 * ctx->sm_count) p.tile *= 2;
  p.tiles = (n + p.tile - 1) / p.tile;
  const size_t list = vtlb_round_up((size_t)n * sizeof(int2), 256);
  void* scr = nullptr;
  if (int rc = ws.get(list + (size_t)p.tiles * 2 * p.cols * 16, &scr)) return rc;
  int2* sorted = (int2*)scr;
  p.sorted = sorted;
  p.partial = (float*)((char*)scr + list);

  VTLB_CUDA(ctx, sort_positions(ctx, ids, n, V, sorted));
  VTLB_LAUNCHED(ctx);

  const unsigned sum_ctas = (unsigned)((p.tiles + p.per_cta - 1) / p.per_cta) * p.slabs;
  auto sums = vec ? (m.any ? embedding_sums_kernel<true, true> : embedding_sums_kernel<true, false>)
                  : (m.any ? embedding_sums_kernel<false, true> : embedding_sums_kernel<false, false>);
  VTLB_CUDA(ctx, vtlb_launch_early(sums, dim3(sum_ctas + zero_ctas), dim3(threads), 0, ctx->stream, p, m, zero_ctas));
  VTLB_LAUNCHED(ctx);
  if (p.tiles > 2) {
    auto join = vec ? embedding_join_kernel<true> : embedding_join_kernel<false>;
    const int wide = (p.cols + 31) / 32, blocks = (p.tiles - 2 + kJoinTiles - 1) / kJoinTiles;
    const int split = wide < 8 ? wide : 8;
    VTLB_CUDA(ctx, vtlb_launch_early(join, dim3((unsigned)blocks * split), dim3(256), 0, ctx->stream, p, split));
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
  const bool y_aligned = vtlb_aligned16(d_Y), vec = D % 4 == 0 && vtlb_aligned16(d_W) && y_aligned;
  // Rows of odd widths in aligned blocks where few warps meet the end of a row (16384 x 4095: 96 -> 90 us, with a mask 139 ->
  // 122; but 16384 x 181: 6.6 -> 7.2).
  const bool blocks_of_w = vtlb_aligned16(d_W) && D >= 512;
  // Four loads in flight per thread where that still leaves eight CTAs for every SM (999 x 2047: one 6.8 us, four 9.3;
  // 3000 x 2047: one 16.1, four 15.3).
  const int U = total >= (size_t)ctx->sm_count * 8 * 256 * 4 * 4 ? 4 : 1;
  auto kern = U == 4 ? (vec ? (m.any ? embedding_fwd_kernel<true, true, 4> : embedding_fwd_kernel<true, false, 4>)
                            : (m.any ? embedding_fwd_kernel<false, true, 4> : embedding_fwd_kernel<false, false, 4>))
                     : (vec ? (m.any ? embedding_fwd_kernel<true, true, 1> : embedding_fwd_kernel<true, false, 1>)
                            : (m.any ? embedding_fwd_kernel<false, true, 1> : embedding_fwd_kernel<false, false, 1>));
  const size_t ctas = (total + 1024 * U - 1) / (1024 * U);
  if (ctas > 0x7fffffffu) return vtlb_fail(ctx, VTLB_EINVAL, "vtlb_embedding_fwd_f32: n * D is beyond 2^43 elements");
  VTLB_CUDA(ctx, vtlb_launch_early(kern, dim3((unsigned)ctas), dim3(256), 0, ctx->stream, (const float*)d_W, V, (uint32_t)D,
                                   (const int32_t*)d_ids_i32, total, scale, (float*)d_Y, blocks_of_w, y_aligned, m, bad));
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
  if (d_src != d_ids_i32 && vtlb_overlap(d_src, n, d_ids_i32, n))
    return vtlb_fail(ctx, VTLB_EINVAL, "vtlb_ids_from_f32: source and ids overlap in part");
  ids_from_f32_kernel<<<grid_for(ctx, n), 256, 0, ctx->stream>>>((const float*)d_src, n, (int32_t*)d_ids_i32);
  VTLB_LAUNCHED(ctx);
  return VTLB_OK;
}
