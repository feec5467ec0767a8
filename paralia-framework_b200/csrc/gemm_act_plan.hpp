// Which variant of the mixed-precision product runs, from sizes and alignment alone (host code without a GPU).
#pragma once
#include <stdint.h>

#include <algorithm>

#include "gemm_act.cuh"

namespace paralia {

constexpr int GA_BK = 64;              // k per stage: 128 bytes, one swizzle row
constexpr int GA_SMS = 148;
// A launch runs one product or two that do not depend on each other: the two of a gradient are then
// one wave of tiles, and one launch.
constexpr int GA_MAX_PROBS = 2;

inline int64_t ga_kblocks(int64_t k) { return (k + GA_BK - 1) / GA_BK; }

// One way to run a product: orientation, tile, split of k.
struct GaPlan {
  bool qc;
  int bn, cg, split;
};

// Estimated microseconds of a variant (a constant common to all is left out). The constants are a fit
// to 3100 timings of 134 shapes (1 to 2048 columns, 300 to 16384 rows, k 256 to 10240) with every
// variant that fits them: the variant it picks is 1.2 % slower than the fastest in the mean, 30 % at
// worst (1024 x 37 x 1024, 6.9 against 5.3 us).
// It knows nothing of columns off 32-byte sectors that are read in place (2888 x 656 x 9320 takes 128 x 128
// tiles, 68 us, where CTA pairs take 58). k is split for tiles of one CTA only; the sum over a cluster is
// written for those.
// Shifts and products in place of most divisions: this is host time of every call (thirty variants, 0.22 us; 1.05 with them).
inline double ga_cost(const GaPlan& v, const int64_t* tiles_of, const int64_t* kblocks, double hbm_bytes, int count) {
  const int log_split = v.split == 1 ? 0 : v.split == 2 ? 1 : v.split == 4 ? 2 : 3;
  int64_t tiles = 0, run = 0, run_sum = 0;
  for (int i = 0; i < count; ++i) {
    const int64_t r = (kblocks[i] + v.split - 1) >> log_split;   // k blocks of a CTA
    tiles += tiles_of[i];
    run_sum += tiles_of[i] * r;
    run = std::max(run, r);
  }
  const double runs = (double)run_sum, mean_run = count == 1 ? (double)run : runs / (double)tiles;
  const int64_t ctas = tiles * v.cg * v.split;
  // CTAs an SM gets: clusters of 4 and 8 do not fill every group of SMs, 36 and 16 fit at a time
  const int64_t share = v.split == 1   ? (ctas + GA_SMS - 1) / GA_SMS
                        : v.split == 2 ? (tiles + 73) / 74
                        : v.split == 4 ? (tiles + 35) / 36
                                       : (tiles + 15) / 16;
  const double turns = (double)(v.bn <= 64 ? (share + 1) >> 1 : share);   // two CTAs an SM, or one
  // a k block: MMAs at 1.4 times BN x 2 clocks, its bytes at 130 GB/s an SM, and 0.23 us from a CTA
  // that runs by itself
  const double bytes = (128.0 + (double)(v.cg == 2 ? v.bn / 2 : v.bn)) * 128.0;
  const double sm = std::max(mean_run * (double)share, (double)run) * std::max(v.bn * (2 / 1900.0 * 1.4), bytes * (1 / 130e3));
  const double alone = std::max(mean_run * turns, (double)run) * 0.23;
  const double in_flight = std::min(1.0, (double)ctas * (1.0 / (2 * GA_SMS)));
  const double hbm = hbm_bytes * (1 / 6.6e6) / (0.88 + 0.12 * in_flight);
  const double l2 = runs * (double)(v.cg * v.split) * bytes * (1 / 15e6);
  return std::max(std::max(sm, alone), std::max(hbm, l2)) + (v.bn * 0.0079) / v.split + (v.qc ? 0.0 : 0.017 * v.bn) +
         (turns - 1.0) * 7.2 * (v.split > 1 ? 1.0 : 0.3) + (v.split > 1 ? 0.18 + 0.039 * v.split + 0.019 * v.bn : 0.0);
}

struct GaChoice {
  GaPlan plan;
  double cost;
};
inline GaChoice ga_choose(const GemmActProblem* ps, int count, bool vec) {
  GaChoice best{{false, 16, 1, 1}, 1e300};
  int64_t kb = INT32_MAX, kblocks[GA_MAX_PROBS], tiles[GA_MAX_PROBS];
  double hbm_bytes = 0.0;
  for (int i = 0; i < count; ++i) {
    const double M = ps[i].M, N = ps[i].N, K = ps[i].K;
    kblocks[i] = ga_kblocks(ps[i].K);
    kb = std::min(kb, std::max<int64_t>(1, kblocks[i]));
    hbm_bytes += 2.0 * (M * K + K * N + M * N);
  }
  for (int qc = vec ? 1 : 0; qc >= 0; --qc) {
    for (int bn = qc ? 64 : 16; bn <= 256; bn = bn < 64 ? bn + 16 : bn * 2) {
      const int cg = bn == 256 ? 2 : 1;
      for (int i = 0; i < count; ++i) {
        const uint32_t R = (uint32_t)(qc ? ps[i].N : ps[i].M), Q = (uint32_t)(qc ? ps[i].M : ps[i].N);
        tiles[i] = (int64_t)((R + 128 * cg - 1) >> (cg == 2 ? 8 : 7)) * ((Q + bn - 1) / (uint32_t)bn);
      }
      for (int split = 1; split <= (bn == 256 ? 1 : 8) && split <= kb; split *= 2) {
        const GaPlan v{qc != 0, bn, cg, split};
        const double c = ga_cost(v, tiles, kblocks, hbm_bytes, count);
        if (c < best.cost) best = {v, c};
      }
    }
  }
  return best;
}

// Fills in the plan of each launch for the products in the order given, and returns how many launches there are.
// Two products go in one launch, which has one plan for both, or one after the other with a plan each:
// the gradient of a few columns is one product with hardly any k and many tiles and one with few tiles
// and much k, which alone is split. 6.2 us of estimate parts them best over 83 shapes: gradient of 16384 x
// 1 x 4096 222 us in one launch and 107 in two, 4096 x 64 x 1024 33 and 23, 4096 x 256 x 4096 44 and 51,
// 2999 x 1000 x 2048 58 and 78.
inline int ga_plan_launches(const GemmActProblem* ps, int n, bool vec, GaPlan* plans) {
  constexpr double second_launch = 6.2;
  const GaChoice both = ga_choose(ps, n, vec);
  plans[0] = both.plan;
  if (n == 1) return 1;
  const GaChoice first = ga_choose(ps, 1, vec), second = ga_choose(ps + 1, 1, vec);
  if (first.cost + second.cost + second_launch >= both.cost) return 1;
  plans[0] = first.plan;
  plans[1] = second.plan;
  return 2;
}

}  // namespace paralia
