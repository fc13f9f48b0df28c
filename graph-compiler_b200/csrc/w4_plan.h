// How a call of the 4-bit linear layer is shared out, and where its pieces lie in shared memory.  Plain C++, so that it can be
// checked without a device.
#pragma once
#include <algorithm>
#include <cstdint>

namespace gcb {

constexpr int kRows = 16;      // outputs of a tile: M of the matrix instruction
constexpr int kBlockK = 128;
constexpr int kCodes = kRows * kBlockK / 2;
constexpr int kW4Warps = 16, kSumWarps = 4, kW4Threads = (kW4Warps + kSumWarps) * 32;
constexpr int kMaxStages = 4;
constexpr int kXPad = 64;            // bytes behind a row of x: neighbouring rows lie 16 banks apart
constexpr int kXMost = 96 * 1024;    // what x may have of a block's shared memory
constexpr int kMostSmem = 223 * 1024;

inline int groups_per_block(int64_t group) { return group >= kBlockK ? 1 : int(kBlockK / group); }
inline int block_bytes(int64_t group, bool zeros) { return kCodes + groups_per_block(group) * kRows * (zeros ? 3 : 2); }

struct W4Plan {
  int pass, nt, rt, cluster, share, wk, clusters, stages;
  int x_at, table_at, meet_at, part_at, smem;
};

inline int up(int v, int step) { return (v + step - 1) / step * step; }

// The fastest way by a model fitted to all ways of twelve shapes.  An SM works off 42 KB of weights a microsecond (near HBM's
// rate), 34 with more than four rows of x and 22 with more than eight, where the products of two instructions' columns and the
// loads of x take most of the issue slots; a warp alone needs 0.15 us for a block.  On top: 15 ns for a turn of the warps, 0.1 us
// for an item, 0.3 where a cluster exchanges its sums, 1 us for a cluster of 2 or 4 and 4 for one of 8 (fewer find room), 8 ns for
// every row and k block of x.  Measured, the plan it takes against the fastest of all: 1 x 28672 x 8192 26.2 us (25.6), 8 rows 34.9
// (31.3), 16 rows 46.2 (44.6); 1 x 4096 x 4096 6.0 (5.9), 16 rows 10.6 (10.4); 5 x 11001 x 4095, groups of 32, 13.7 (13.5).
inline bool plan_w4(int M, int tiles, int kblocks, int gpb, int bytes, const int *at_once, W4Plan *best) {
  double cost = 1e30;
  for (int pass = std::min(M, 16); pass >= 1 && cost == 1e30; pass = pass > 8 ? 8 : pass / 2) {   // fewer rows at a time only where x does not fit
    const int nt = pass > 8 ? 2 : 1;
    for (int cluster = 1; cluster <= 8; cluster *= 2) {
      const int share = (kblocks + cluster - 1) / cluster;
      // in 64 bits: a plan whose sizes have wrapped would be taken for one that fits
      if (at_once[cluster] < 1 || cluster > kblocks || (pass + 1) * (int64_t(share) * kBlockK * 2 + kXPad) > kXMost) continue;
      for (int rt = 1; rt <= 2; ++rt)
        for (int wk = 1; wk <= kW4Warps; wk *= 2) {
          const int per_item = rt * (kW4Warps / wk), items = (tiles + per_item - 1) / per_item;
          W4Plan p{pass, nt, rt, cluster, share, wk, std::min(at_once[cluster], items), 0, 0, 0, 0, 0, 0};
          const int outs = 16 * per_item, turns = (share + wk - 1) / wk, most = (tiles + p.clusters - 1) / p.clusters;
          const int x = up((pass + 1) * (share * kBlockK * 2 + kXPad), 128), table = up((pass + 1) * share * gpb * 8, 128);
          const int meet = up(kW4Warps * 8 * nt * (16 * rt + 4) * 4, 128), part = cluster > 1 ? 2 * 8 * nt * outs * 4 : 0;
          const int stage = kW4Warps * rt * bytes, room = (kMostSmem - x - table - meet - part) / stage;
          if (room < 2) continue;
          p.stages = std::min(kMaxStages, room);
          p.x_at = up(p.stages * stage, 128);
          p.table_at = p.x_at + x;
          p.meet_at = p.table_at + table;
          p.part_at = p.meet_at + meet;
          p.smem = p.part_at + part;
          const double rate = (pass > 8 ? 22e3 : pass > 4 ? 34e3 : 42e3) * (rt == 2 && pass > 2 ? 0.96 : 1.0);   // two tiles at a time: fewer registers to spare
          const int full = most / per_item, rest = most - full * per_item;
          const double us = turns * (double(full) * per_item * wk * bytes / rate + (rest ? std::max(rest * wk * bytes / rate, rt * 0.15) : 0.0)) +
                            (full + (rest > 0)) * ((cluster > 1 ? 0.3 : 0.1) + 0.015 * turns) + (cluster > 4 ? 4.0 : cluster > 1 ? 1.0 : 0.0) + 0.008 * pass * share;
          if (us < cost) {
            cost = us;
            *best = p;
          }
        }
    }
  }
  return cost < 1e30;
}

} // namespace gcb
