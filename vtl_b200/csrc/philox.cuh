// The counter-based generator behind dropout: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", SC 2011).  Element i of call `step` under key `seed` draws word i % 4 of the block whose 128-bit
// counter is (i / 4, step), so a mask is a pure function of (seed, step, i): the backward pass computes it again
// instead of reading it, a fused kernel and a pass of its own agree, and no launch geometry shows in it.  The
// initialisers' generator (init.cu) is not used here: its seeds of neighbouring layers are neighbouring states of one
// sequence, which is harmless for weights drawn once and not for masks drawn every step.
#pragma once
#include "common.cuh"

// An element is dropped when its word is below floor(p * 2^32), that is at most `last`; kept ones are multiplied by
// `keep`.  With p below 2^-32 nothing is dropped and keep rounds to 1: `any` is false and the callers draw no words.
// With p = 1 every word is at most `last`.
struct vtlb_mask {
  uint32_t last;
  float keep;  // 1 / (1 - p), rounded once
  uint32_t key0, key1, step0, step1;
  bool any;
};

inline vtlb_mask vtlb_make_mask(double p, uint64_t seed, uint64_t step) {
  vtlb_mask m;
  const uint64_t below = (uint64_t)(p * 4294967296.0);
  m.any = below > 0;
  m.last = (uint32_t)(below - 1);
  m.keep = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
  m.key0 = (uint32_t)seed, m.key1 = (uint32_t)(seed >> 32);
  m.step0 = (uint32_t)step, m.step1 = (uint32_t)(step >> 32);
  return m;
}

#ifdef __CUDACC__
__device__ __forceinline__ uint4 vtlb_philox(const vtlb_mask& m, uint64_t block) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = m.step0, c3 = m.step1;
  uint32_t k0 = m.key0, k1 = m.key1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// A dropped element is zero whatever it held, NaN and infinities included.
__device__ __forceinline__ float vtlb_drop(const vtlb_mask& m, uint32_t word, float x) {
  return word > m.last ? __fmul_rn(x, m.keep) : 0.0f;
}
__device__ __forceinline__ float4 vtlb_drop4(const vtlb_mask& m, uint64_t block, float4 v) {
  const uint4 r = vtlb_philox(m, block);
  return make_float4(vtlb_drop(m, r.x, v.x), vtlb_drop(m, r.y, v.y), vtlb_drop(m, r.z, v.z), vtlb_drop(m, r.w, v.w));
}
#endif
