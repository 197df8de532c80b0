// qmlp_mx_plan.hip -- how an MXFP4 product runs for its sizes (host code).
#include "qmlp_internal.h"
#include "qmlp_mx.h"

namespace qmlp {

// Every candidate's time in microseconds, linear in what it does, and the cheapest one wins.  The
// constants were fitted (non-negative least squares on the relative error) to 4600 measured (sizes,
// candidate) points on 256 CUs: 16 shapes from N = 96 to 17408 and K = 512 to 17408 with one and two
// matrices, 8 to 2048 tokens.  The plan they pick was on average 2 % slower than the fastest measured
// candidate of all that were built then (more stream variants among them), at worst 36 % (10.1 against
// 7.4 us, where streamed and tiled kernels meet).
//
// Streamed, per workgroup: launch and tail; units of K a wave takes in turn; all (32 features x token
// group x unit) products of the launch and all weight units it reads, per CU; rounds of workgroups.
struct StreamCost {
  int waves, groups;  // token groups of 32 a workgroup
  double start, unit, product, weight, round;
};
constexpr StreamCost kStreamCost[2][3] = {
    {{4, 1, 0.96, 0.937, 0.078, 0.164, 0.179}, {8, 1, 0.97, 0.701, 0.119, 0.070, 0.720}, {8, 2, 0.22, 1.160, 0.155, 0.048, 1.507}},
    {{4, 1, 2.09, 0.987, 0.131, 0.256, 0.133}, {8, 1, 0.76, 0.770, 0.173, 0.289, 1.389}, {4, 2, 0.70, 0.616, 0.155, 0.370, 2.751}}};
// Tiled: launch; a tile's start and end; a unit of K of a tile, alone on its CU and by how many CUs are
// busy (the shared power and bandwidth: a full machine takes half as long again), of which the weights'
// part falls with the token blocks that share them; the sum launch and a MB of partial tiles.
struct TileCost {
  double start, round, unit, busy, weight, sum, mbyte;
};
constexpr TileCost kTileCost[2][4] = {
    {{3.92, 0.217, 0.435, 0.232, 0.087, 2.56, 0.326}, {5.27, 0.170, 0.493, 0.352, 0.0, 1.96, 0.410},
     {3.99, 2.190, 0.681, 0.499, 0.0, 2.08, 0.309}, {0.0, 6.876, 0.938, 0.472, 0.0, 2.01, 0.292}},
    {{2.18, 1.665, 0.348, 0.314, 0.649, 5.35, 0.205}, {3.04, 1.997, 0.421, 0.622, 0.356, 3.69, 0.276},
     {1.99, 3.779, 0.630, 0.744, 0.170, 3.78, 0.259}, {0.0, 6.770, 0.884, 0.695, 0.0, 4.76, 0.293}}};
constexpr int kPieces[] = {1, 2, 3, 4, 6, 8, 12};
constexpr int kMostStreamed = 1024;  // tokens: beyond, the tiles win at every measured shape

MxPlan mx_plan(int M, int N, int K, int nmat, int num_cus) {
  const double cus = num_cus;
  const long nsb = mx_ksb(K), rows = mx_row_tiles(N);
  auto up = [](long a, long b) { return (a + b - 1) / b; };
  MxPlan best{kMxStream, 0, 1, 0, 0};
  double best_us = 1e30;
  if (M <= kMostStreamed) {
    for (int v = 0; v < 3; ++v) {
      const StreamCost& c = kStreamCost[nmat - 1][v];
      const long ty = up(M, 32 * c.groups);
      const double us = c.start + c.unit * up(nsb, c.waves) + c.product * (double)(rows * ty * nsb) / cus +
                        c.weight * (double)(rows * nsb) / cus + c.round * up(rows * ty, num_cus);
      if (us < best_us && (v < 2 || M > 32)) {
        best_us = us;
        best = MxPlan{v == 0 ? kMxStream : v == 1 ? kMxStreamLong : kMxStreamWide, 0, 1, (int)(rows * ty), 0};
      }
    }
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

// Whether the streamed product quantises unpacked rows by itself, every workgroup all of them.
bool mx_quantizes_inside(int M, int K) { return M <= kMxInside && (size_t)mx_ksb(K) * M * 136 <= 40960; }

}  // namespace qmlp
