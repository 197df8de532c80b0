// qmlp_mx_plan.hip -- how an MXFP4 product runs for its sizes (host code).
#include "qmlp_internal.h"
#include "qmlp_mx.h"

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

MxPlan mx_plan(int M, int N, int K, int nmat, int num_cus) {
  const double cus = num_cus;
  const long nsb = mx_ksb(K), rows = mx_row_tiles(N);
  auto up = [](long a, long b) { return (a + b - 1) / b; };
  MxPlan best{kMxStream, 0, 1, 0, 0};
  double best_us = 1e30;
  auto streamed = [&](const StreamCost& c) {
    const long ty = up(M, 32 * c.groups);
    const double us = c.start + c.unit * up(nsb, c.waves) + c.product * (double)(rows * ty * nsb) / cus +
                      c.weight * (double)(rows * nsb) / cus + c.round * up(rows * ty, num_cus);
    if (us < best_us && M > 32 * (c.groups - 1)) {
      best_us = us;
      best = MxPlan{c.kind, 0, 1, (int)(rows * ty), 0};
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
        best = MxPlan{kMxTiles, h, ks, (int)pieces, bytes};
      }
    }
  }
  return best;
}

// Whether the streamed product quantises unpacked rows by itself, every workgroup all of them, rather than
// leaving it to a launch in front.  Inside / in front, us: one token 12.1 / 13.6 at 5120 x 17408, 10.7 /
// 13.6 at 17408 x 5120, 19.6 / 21.4 for two such matrices, 4.1 / 5.5 at 2048 x 2048; two tokens of K = 17408
// 13.5 / 13.6, three 14.9 / 13.6; four tokens of K = 5120 13.7 / 14.9, for two matrices 21.8 / 21.5.
bool mx_quantizes_inside(int M, int K) { return M <= kMxInside && mx_ksb(K) * M <= 136; }

}  // namespace qmlp
