// How group norm cuts its work (groupnorm.cu); plain C++, so that it can be checked for every size without a GPU.
#pragma once
#include <climits>

// Channels are taken in slabs of whole groups.  A thread-block cluster owns one slab of one sample; its CTAs cut the
// positions into `rsplit` equal stretches (and a slab too wide for the threads of one CTA into `csplit` pieces), and
// each CTA keeps its piece in registers: `vpt` pieces of `vec` channels a thread.
struct GnPlan {
  bool on_chip;     // false: the group does not fit a cluster's registers; x is read twice
  int vec;          // channels per load: 4 (16-byte aligned rows) or 1
  int vpt;          // rows per thread: 1, the middle or the largest number that the kernel at hand has
  int groups;       // per slab; the last slab may have fewer
  int slabs;
  int csplit, rsplit;
  int channels;     // per CTA (a multiple of vec), the last piece of a slab may have fewer
  int rows;         // per CTA, the last stretch may have fewer
  bool tma;         // the pieces are fetched by TMA, in `boxes` boxes of `box_rows` rows (a multiple of eight) each
  int boxes, box_rows;
};

constexpr int kGnFwdThreads = 512, kGnBwdThreads = 256, kGnMaxGroups = 32, kGnMaxCluster = 8;
constexpr int kGnMaxChannels = INT_MAX - 1023;  // a CTA's channels, up to 1024, are rounded up and counted in ints
constexpr int kGnMaxSmem = 150 << 10;  // for the pieces; with the kernels' static arrays within 227 KB

// The kernels have `middle` and `most` rows per thread to choose from, and one; a row's pieces take a power of two of the
// threads.
inline int gn_pow2(int n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

// The plan with `groups` groups per slab.
inline GnPlan gn_plan_slab(int B, int S, int C, int G, int vec, int groups, int threads, int middle, int most, int sm_count) {
  GnPlan p = {};
  p.vec = vec;
  p.groups = groups;
  p.slabs = (G + groups - 1) / groups;
  const int cols = groups * (C / G) / vec;
  p.csplit = 1;
  while ((cols + p.csplit - 1) / p.csplit > threads && p.csplit < kGnMaxCluster) p.csplit *= 2;
  const int cols_cta = (cols + p.csplit - 1) / p.csplit;
  p.channels = cols_cta * vec;
  if (cols_cta > threads || groups > kGnMaxGroups) return p;
  const int lanes = threads / gn_pow2(cols_cta);  // rows that a CTA takes in one step
  const auto fits = [&](int vpt, int rsplit) { return (long long)lanes * vpt * rsplit >= S; };
  const int max_r = kGnMaxCluster / p.csplit;
  p.rsplit = 1;
  while (p.rsplit < max_r && !fits(most, p.rsplit)) ++p.rsplit;
  if (!fits(most, p.rsplit)) return p;
  // Too few CTAs for the SMs: shorter stretches.
  while (p.rsplit * 2 <= max_r && !fits(1, p.rsplit) && (long long)B * p.slabs * p.csplit * p.rsplit * 2 <= sm_count) p.rsplit *= 2;
  p.rows = (S + p.rsplit - 1) / p.rsplit;
  p.vpt = p.rows <= lanes ? 1 : p.rows <= lanes * middle ? middle : most;
  // TMA boxes are at most 256 by 256; rows of less than 64 bytes are not worth one.  Nor is a map, half a microsecond of the
  // host's time, for a few pieces of one step (8 x 8 positions of 128 channels: 7.1 us a call with one, 6.6 us without).
  const bool few = p.vpt == 1 && (long long)B * p.slabs * p.csplit * p.rsplit <= 2LL * sm_count;
  p.tma = vec == 4 && p.channels >= 16 && p.channels <= 256 && !few;
  p.boxes = (p.rows + 255) / 256;
  p.box_rows = ((p.rows + p.boxes - 1) / p.boxes + 7) / 8 * 8;
  p.on_chip = true;
  return p;
}

inline GnPlan gn_plan(int B, int S, int C, int G, bool aligned, int threads, int middle, int most, int sm_count) {
  const int width = C / G, vec = aligned && C % 4 == 0 ? 4 : 1;
  int unit = 1;  // groups whose channels are a multiple of vec
  while (((long long)unit * width) % vec) ++unit;
  // Slabs of 32 channels and more (128-byte pieces of a row) up to 32 pieces a row, the one that wastes fewest threads;
  // narrower ones for groups that do not fit otherwise.
  GnPlan best = {};
  double best_score = -1.0;
  for (int groups = unit; groups == unit || (groups <= G && (long long)groups * width <= 32 * vec); groups += unit) {
    const int k = groups < G ? groups : G;
    if (k > kGnMaxGroups && k > unit) break;
    const GnPlan p = gn_plan_slab(B, S, C, G, vec, k, threads, middle, most, sm_count);
    const int cols = p.channels / vec, channels = k * width;
    const double score = (p.on_chip ? 4.0 : 0.0) + (channels >= 32 || k == G ? 2.0 : channels / 32.0) + (double)cols / gn_pow2(cols);
    if (score > best_score + 1e-9) best = p, best_score = score;
    if (score >= 7.0) break;  // there is no better one
  }
  return best;
}
