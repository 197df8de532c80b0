// qmlp_mx_plan.hip -- how an MXFP4 product runs for its sizes (host code).
#include "qmlp_internal.h"
#include "qmlp_mx8.h"

namespace qmlp {

// Every candidate's time in microseconds, linear in what it does, and the cheapest one wins.  The
// constants were fitted (non-negative least squares, points near the fastest of their sizes weighing
// most) to 5900 measured (sizes, candidate) points on 256 CUs with packed activations: 16 shapes from N = 96
// to 17408 and K = 512 to 17408 with one and two matrices, 21 token counts from 8 to 2048 (for the streamed
// kernels the points of matrices beyond 40 million values weigh six times).  Measured again on the kernels
// as they are, up to 1024 tokens the plan is on average 2.1 % (one matrix) and 1.4 % (two) slower than the
// fastest measured candidate, at worst 25 % (9.4 against 7.5 us at 96 tokens of 3000 x 5120, where streamed
// and tiled kernels meet).
//
// Streamed, per workgroup: launch and tail; units of K a wave takes in turn; all (32 features x token
// group x unit) products of the launch and all weight units it reads, per CU; rounds of workgroups.
struct StreamCost {
  MxKind kind;
  int waves, groups;  // token groups of 32 a workgroup
  double start, unit, product, weight, round;
};
constexpr StreamCost kStreamCost[] = {{kMxStream, 4, 1, 1.15, 0.982, 0.062, 0.125, 0.187},
                                      {kMxStreamDeep, 4, 1, 1.92, 0.343, 0.115, 0.066, 0.235},
                                      {kMxStreamLong, 8, 1, 1.22, 0.461, 0.133, 0.029, 1.022},
                                      {kMxStreamWide, 8, 2, 0.0, 0.862, 0.174, 0.006, 2.188}};
constexpr StreamCost kPairCost[] = {{kMxStream, 4, 1, 2.26, 0.739, 0.222, 0.140, 0.0},
                                    {kMxStreamLong, 8, 1, 0.76, 0.685, 0.252, 0.159, 1.407},
                                    {kMxStreamWide, 4, 2, 0.20, 0.558, 0.219, 0.257, 3.209}};
// Tiled: launch; a tile's start and end; a unit of K of a tile, alone on its CU, and by how many CUs are
// busy with tokens (the shared power and bandwidth: on a full machine a unit takes 1.4 to 2.6 times as
// long); the weights' part, which falls with the token blocks that share them; the sum launch and a MB
// of partial tiles.
struct TileCost {
  double start, round, unit, busy, weight, sum, mbyte;
};
constexpr TileCost kTileCost[2][4] = {
    {{2.72, 1.699, 0.412, 0.207, 0.161, 3.18, 0.229}, {2.25, 3.522, 0.415, 0.430, 0.126, 2.64, 0.241},
     {3.24, 3.465, 0.483, 0.869, 0.0, 0.0, 0.0}, {0.0, 7.281, 0.663, 1.031, 0.0, 0.0, 0.0}},
    {{1.50, 2.410, 0.378, 0.250, 0.499, 4.19, 0.169}, {1.25, 3.590, 0.394, 0.505, 0.522, 3.70, 0.217},
     {1.78, 3.979, 0.476, 0.916, 0.296, 0.0, 0.0}, {0.59, 5.642, 0.638, 1.219, 0.218, 0.0, 0.0}}};
// Tiles of more than two heights stay whole: split, they won nowhere.
constexpr int kMostSplit = 2;
constexpr int kPieces[] = {1, 2, 3, 4, 6, 8, 12};
// Tokens up to which the streamed kernels are candidates.  Beyond, the tiles win at 15 of the 16 measured
// shapes; at the narrowest, 96 x 5120, streaming took 4.2 us at 2048 tokens and the planned tiles take 10.1.
constexpr int kMostStreamed = 1024;

static MxPlan plan_a8(int M, int N, int K, int nmat, int num_cus);

MxPlan mx_plan(int M, int N, int K, int nmat, int num_cus, bool a8) {
  if (a8) return plan_a8(M, N, K, nmat, num_cus);
  const double cus = num_cus;
  const long nsb = mx_ksb(K), rows = mx_row_tiles(N);
  auto up = [](long a, long b) { return (a + b - 1) / b; };
  MxPlan best{kMxStream, 0, 1, 0, 0, 0};
  double best_us = 1e30;
  auto streamed = [&](const StreamCost& c) {
    const long ty = up(M, 32 * c.groups);
    const double us = c.start + c.unit * up(nsb, c.waves) + c.product * (double)(rows * ty * nsb) / cus +
                      c.weight * (double)(rows * nsb) / cus + c.round * up(rows * ty, num_cus);
    if (us < best_us && M > 32 * (c.groups - 1)) {
      best_us = us;
      best = MxPlan{c.kind, 0, 1, (int)(rows * ty), 0, 0};
    }
  };
  if (M <= kMostStreamed) {
    if (nmat == 1)
      for (const StreamCost& c : kStreamCost) streamed(c);
    else
      for (const StreamCost& c : kPairCost) streamed(c);
  }
  if (M <= kMxFewTokens) return best;
  for (int h = 1; h <= 4; ++h) {
    const TileCost& c = kTileCost[nmat - 1][h - 1];
    const long ntt = up(M, 64 * h), tiles = up(N, 256 / nmat) * ntt;
    const double filled = (double)up(M, 32) / (double)(ntt * 2 * h);  // token units that hold tokens
    for (int ks : kPieces) {
      if (ks > nsb || (ks > 1 && h > kMostSplit)) break;
      const long pieces = tiles * ks, full = pieces / num_cus, rest = pieces % num_cus, units = up(nsb, ks);
      const size_t bytes = ks > 1 ? (size_t)pieces * 256 * 64 * h * 4 : 0;
      if (bytes > kMxPartBytes) break;
      const double turns = full + (rest ? 1 : 0), busy = full + rest / cus;
      const double us = c.start + c.round * turns +
                        units * (c.unit * turns + c.busy * busy * filled + c.weight * busy / ntt) +
                        (ks > 1 ? c.sum + c.mbyte * (double)bytes * 1e-6 * filled : 0.0);
      if (us < best_us) {
        best_us = us;
        best = MxPlan{kMxTiles, h, ks, (int)pieces, bytes, 0};
      }
    }
  }
  return best;
}

// The same for 8-bit activations and more than 16 tokens, in tiles of two heights (the streamed kernels with one unit
// of K under way, but for kMxStreamDeep with two), fitted the same way to 5366 points of 10 shapes from N = 96 to 17408
// and K = 512 to 17408 at 22 token counts: 0.9 % slower on average than the fastest measured candidate, at worst 17 %
// (11.9 against 10.1 us at 777 tokens of 1000 x 2976).  What full rounds of tiles leave over may run in pieces by
// itself: 2048 tokens of 17408 -> 5120, 320 tiles on 256 CUs, took 218.6 us in whole tiles and take 178.7 with 64 tiles
// in four pieces behind 256 whole ones.
constexpr StreamCost kStreamCost8[] = {{kMxStream, 4, 1, 3.389, 0.609, 0.138, 0.127, 0.119},
                                       {kMxStreamDeep, 4, 1, 3.597, 0.409, 0.174, 0.050, 0.551},
                                       {kMxStreamLong, 8, 1, 3.615, 0.676, 0.171, 0.098, 0.101},
                                       {kMxStreamWide, 8, 2, 3.225, 1.142, 0.244, 0.143, 0.633}};
constexpr StreamCost kPairCost8[] = {{kMxStream, 4, 1, 2.747, 1.494, 0.181, 0.181, 0.353},
                                     {kMxStreamLong, 8, 1, 3.185, 1.359, 0.222, 0.155, 0.785}};
constexpr TileCost kTileCost8[2][2] = {
    {{3.55, 2.655, 0.581, 0.528, 0.609, 2.44, 0.152}, {3.83, 3.971, 0.683, 1.108, 0.311, 1.68, 0.208}},
    {{3.98, 2.667, 0.608, 0.516, 0.318, 3.54, 0.163}, {3.83, 4.025, 0.712, 1.105, 0.115, 3.18, 0.192}}};

static MxPlan plan_a8(int M, int N, int K, int nmat, int num_cus) {
  const double cus = num_cus;
  const long nsb = mx_ksb(K), rows = mx_row_tiles(N);
  auto up = [](long a, long b) { return (a + b - 1) / b; };
  if (M <= kMx8FewTokens) return MxPlan{kMxFew, rows > num_cus ? 4 : 8, 1, (int)rows, 0, 0};
  MxPlan best{kMxStream, 0, 1, 0, 0, 0};
  double best_us = 1e30;
  auto streamed = [&](const StreamCost& c) {
    const long ty = up(M, 32 * c.groups);
    const double us = c.start + c.unit * up(nsb, c.waves) + c.product * (double)(rows * ty * nsb) / cus +
                      c.weight * (double)(rows * nsb) / cus + c.round * up(rows * ty, num_cus);
    if (us < best_us && M > 32 * (c.groups - 1)) {
      best_us = us;
      best = MxPlan{c.kind, 0, 1, (int)(rows * ty), 0, 0};
    }
  };
  if (M <= kMostStreamed) {
    if (nmat == 1)
      for (const StreamCost& c : kStreamCost8) streamed(c);
    else
      for (const StreamCost& c : kPairCost8) streamed(c);
  }
  if (M <= kMxFewTokens) return best;
  for (int h = 1; h <= 2; ++h) {
    const TileCost& c = kTileCost8[nmat - 1][h - 1];
    const long ntt = up(M, 64 * h), tiles = up(N, 256 / nmat) * ntt;
    const double filled = (double)up(M, 32) / (double)(ntt * 2 * h);  // token units that hold tokens
    const long most = tiles / num_cus * num_cus;
    for (long whole : {0l, most}) {
      for (int ks : kPieces) {
        if (whole && (whole == tiles || ks == 1)) continue;  // the same as none
        if (ks > nsb) break;
        const long pieces = (tiles - whole) * ks, rest = pieces % num_cus, units = up(nsb, ks);
        const size_t bytes = ks > 1 ? (size_t)pieces * 256 * 64 * h * 4 : 0;
        if (bytes > kMxPartBytes) break;
        const double first = whole / cus, turns = up(pieces, num_cus), busy = pieces / num_cus + rest / cus;
        const double unit_turns = units * turns + nsb * first, unit_busy = units * busy + nsb * first;
        const double us = c.start + c.round * (turns + first) + c.unit * unit_turns + c.busy * unit_busy * filled +
                          c.weight * unit_busy / ntt + (ks > 1 ? c.sum + c.mbyte * (double)bytes * 1e-6 * filled : 0.0);
        if (us < best_us) {
          best_us = us;
          best = MxPlan{kMxTiles, h, ks, (int)(whole + pieces), bytes, (int)whole};
        }
      }
    }
  }
  return best;
}

// Whether the streamed product quantises unpacked rows by itself, every workgroup all of them, rather than
// leaving it to a launch in front.  Inside / in front, us: one token 12.1 / 13.6 at 5120 x 17408, 10.7 /
// 13.6 at 17408 x 5120, 19.6 / 21.4 for two such matrices, 4.1 / 5.5 at 2048 x 2048; two tokens of K = 17408
// 13.5 / 13.6, three 14.9 / 13.6; four tokens of K = 5120 13.7 / 14.9, for two matrices 21.8 / 21.5.  8-bit activations
// (the few-token kernel), captured, eight matrices in turn: one token 3.6 / 5.7 at 2048 x 2048, 11.6 / 14.7 at 17408 x
// 5120 (N x K), 13.2 / 18.4 at 5120 x 17408, 18.9 / 22.8 for two of 17408 x 5120; three tokens of K = 5120 (60 units)
// 7.1 / 8.3 at N = 5120, 13.8 / 14.1 at 17408, two matrices 20.5 / 21.6; two of K = 8704 (68) 9.4 / 10.9.  Beyond, either
// may win: four of K = 5120 (80) 7.9 / 8.4, 15.5 / 13.8 and 21.0 / 21.4; of K = 8704 three (102) 10.1 / 10.6, four (136)
// 11.3 / 10.5.
bool mx_quantizes_inside(int M, int K, bool a8) { return M <= kMxInside && mx_ksb(K) * M <= (a8 ? 68 : 136); }

}  // namespace qmlp
