// qmlp_xcd.h -- which block of a launch takes which tile, shared by the many-token kernels.
#pragma once

namespace qmlp {

// The tile (or piece) of block b among P, so that each XCD (block b runs on XCD b % 8) takes one
// contiguous run of them, P / 8 or one more, whatever P is: neighbours share weights, or a split
// tile's partial tiles, in its L2.  With the runs only where P is a multiple of 8 and block order
// elsewhere, every XCD read every weight: bf16 gate/up of 4608 x 6400 at 259 tokens, 250 tiles,
// 81.8 us, with them 42.0; a count of 748 tiles at the 27B shape, bound by its products, 427.7 and
// 427.3.
__host__ __device__ constexpr int xcd_run(int b, int P) {
  return b % 8 * (P / 8) + (b % 8 < P % 8 ? b % 8 : P % 8) + b / 8;
}
constexpr bool xcd_runs_are_contiguous(int P) {
  int expect = 0;
  for (int x = 0; x < 8; ++x)
    for (int b = x; b < P; b += 8)
      if (xcd_run(b, P) != expect++) return false;
  return expect == P;
}
static_assert(xcd_runs_are_contiguous(1) && xcd_runs_are_contiguous(250) && xcd_runs_are_contiguous(255) &&
              xcd_runs_are_contiguous(256) && xcd_runs_are_contiguous(748));

}  // namespace qmlp
