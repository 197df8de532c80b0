// qmlp_mx_plan.hip -- how an MXFP4 product runs for its sizes (host code).
#include "qmlp_internal.h"
#include "qmlp_mx.h"

namespace qmlp {

// Every candidate's time in microseconds, linear in what it does, and the cheapest one wins.  The
// constants were fitted (non-negative least squares on the relative error) to 4600 measured (sizes,
// candidate) points on 256 CUs: 16 shapes from N = 96 to 17408 and K = 512 to 17408 with one and two
// matrices, 8 to 2048 tokens.  The plan they pick was on average 2.5 % (one matrix) and 1.3 % (two) slower
// than the fastest measured one, at worst 32 % (10.0 against 7.6 us at 128 tokens of 3000 x 5120, where
// streamed and tiled kernels meet).
//
// Streamed, per workgroup: launch and tail; units of K a wave takes in turn; all (32 features x token
// group x unit) products of the launch and all weight units it reads, per CU; rounds of workgroups.
struct StreamCost {
  MxKind kind;
  int waves, groups;  // token groups of 32 a workgroup
  double start, unit, product, weight, round;
};
constexpr StreamCost kStreamCost[] = {{kMxStream, 4, 1, 1.41, 0.861, 0.076, 0.182, 0.142},
                                      {kMxStreamDeep, 4, 1, 1.47, 0.518, 0.085, 0.102, 0.303},
                                      {kMxStreamLong, 8, 1, 1.07, 0.739, 0.112, 0.079, 0.728},
                                      {kMxStreamWide, 8, 2, 0.39, 1.158, 0.154, 0.043, 1.482}};
constexpr StreamCost kPairCost[] = {{kMxStream, 4, 1, 2.36, 0.920, 0.118, 0.268, 0.149},
                                    {kMxStreamLong, 8, 1, 1.05, 0.668, 0.163, 0.308, 1.359},
                                    {kMxStreamWide, 4, 2, 0.96, 0.519, 0.148, 0.393, 2.707}};
// Tiled: launch; a tile's start and end; a unit of K of a tile, alone on its CU and by how many CUs are
// busy (the shared power and bandwidth: on a full machine a unit takes half as long again), of which the
// weights' part falls with the token blocks that share them; the sum launch and a MB of partial tiles.
struct TileCost {
  double start, round, unit, busy, weight, sum, mbyte;
};
constexpr TileCost kTileCost[2][4] = {
    {{4.10, 0.171, 0.408, 0.197, 0.117, 2.65, 0.319}, {4.99, 0.540, 0.456, 0.307, 0.0, 2.46, 0.320},
     {3.80, 2.460, 0.640, 0.372, 0.0, 2.66, 0.256}, {0.0, 6.968, 0.870, 0.400, 0.0, 3.16, 0.232}},
    {{1.97, 1.892, 0.360, 0.227, 0.685, 5.20, 0.177}, {2.59, 2.480, 0.436, 0.379, 0.454, 3.86, 0.239},
     {2.16, 3.695, 0.633, 0.506, 0.150, 4.04, 0.224}, {0.0, 6.789, 0.870, 0.494, 0.0, 4.10, 0.262}}};
constexpr int kPieces[] = {1, 2, 3, 4, 6, 8, 12};
constexpr int kMostStreamed = 1024;  // tokens: beyond, the tiles win at every measured shape

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
    for (int ks : kPieces) {
      if (ks > nsb) break;
      const long pieces = tiles * ks, full = pieces / num_cus, rest = pieces % num_cus, units = up(nsb, ks);
      const size_t bytes = ks > 1 ? (size_t)pieces * 256 * 64 * h * 4 : 0;
      if (bytes > kMxPartBytes) break;
      const double turns = full + (rest ? 1 : 0), busy = full + rest / cus;
      const double us = c.start + c.round * turns + units * (c.unit * turns + c.busy * busy + c.weight * busy / ntt) +
                        (ks > 1 ? c.sum + c.mbyte * (double)bytes * 1e-6 : 0.0);
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
