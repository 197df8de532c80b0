// qmlp_mx_stream.hip -- MXFP4 products of few tokens: one workgroup per 32 features x 32 (or 64) tokens
// (layout: qmlp_mx.h).
//
// Bound by the weights: 17/32 byte each, read once.  A lane's 16-byte load is an operand of the scaled
// 32x32x64 product as it comes, so a wave does nothing but load and multiply (a CU's matrix cores could
// take 128 B a cycle, its share of the memory is 13), and one or two K units (4352 B of each matrix) a
// wave, 5 to 9 waves a CU, keep 11-19 MB under way on the card.  With M <= 4 (and few enough values) x is
// quantised by the workgroups themselves, which saves a launch.  Weights pass the caches by
// (non-temporal): eight layers' in turn, 47 MB each, take 11.4 us instead of 12.0; three, which the
// memory-side cache holds, 11.1 instead of 9.2.
// Measured (eight matrices in turn): 5120 x 17408 one token 11.4 us (4.2 TB/s), 17408 x 5120 16 tokens
// 11.9 (4.0 TB/s), two of them one token 19.4 (4.9 TB/s); reading the same bytes and nothing else takes
// 8.7 and 15.7 us.  The token operands come from the L2 with the weights' loads; staged in LDS first they
// cost 0.7 us less at 5120 x 17408 and one token, and 1.7 to 4 us more at 17408 x 5120 and 16.  Half units
// as the waves' steps, which share K out more evenly, read the scales twice: 12.8-14.2 us for 11.5.
#include <type_traits>

#include "qmlp_internal.h"
#include "qmlp_mx8.h"

namespace qmlp {

// One 256-K unit of N 32-row matrices: the lane's 16 code bytes of the four K-steps and the dword with
// their scales.
template <int N>
struct MxStage {
  i32x4 code[N][4];
  uint32_t scale[N];
};

// The same of MG token groups with 8-bit activations: both planes of a lane's blocks.
template <int MG>
struct Mx8Stage {
  i32x4 plane[MG][4][2];
  uint32_t scale[MG];
};

// out^T[features, tokens] = W x^T: the weights as the A operand, MG groups of 32 token rows as B.  The
// waves of a workgroup share the units of K out in turn, so that it reads every weight matrix front to
// back, and add their sums up in a fixed order through LDS (deterministic).  A8: 8-bit activations, whose lanes
// make two operands of a plane pair (some 24 bit operations to two products): 17 to 32 tokens of 17408 -> 5120 take
// 18.5-19.7 us, of the pair 5120 -> 17408 26 (up to 16, in their own kernel, 13.7 and 21).
template <int NMAT, int WAVES, int MG, int D, int MODE, int XT, bool A8>
__global__ __launch_bounds__(WAVES * 64) void mx_stream_kernel(const uint8_t* __restrict__ x,
                                                              const uint8_t* __restrict__ w0,
                                                              const uint8_t* __restrict__ w1, int nsb, MxOut o,
                                                              int K, size_t row_bytes) {
  constexpr int kRow = 36;  // floats a token's 32 features take in LDS
  constexpr int kHalfWaves = WAVES / 2;
  __shared__ float s_part[NMAT][MG][kHalfWaves][32 * kRow];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ft = blockIdx.x, tt0 = blockIdx.y * MG, half = lane >> 5;
  const uint8_t* wp[2] = {w0 + (size_t)ft * nsb * kMxUnit, NMAT > 1 ? w1 + (size_t)ft * nsb * kMxUnit : nullptr};
  // token rows behind the last one read it again
  const uint8_t* xp[MG];
  uint32_t boff[MG];
#pragma unroll
  for (int g = 0; g < MG; ++g) {
    const int tt = min(tt0 + g, (o.M - 1) / 32);
    xp[g] = x + (size_t)tt * nsb * (A8 ? kMx8Unit : kMxUnit);
    boff[g] = half * 32 + min(lane & 31, o.M - 1 - tt * 32);
  }
  constexpr bool kInside = XT != kMxPackedX;
  static_assert(!(kInside && A8), "few rows in 8 bits are the few-token kernel's");
  using Tokens = std::conditional_t<A8, Mx8Stage<MG>, MxStage<MG>>;
  extern __shared__ __align__(16) uint8_t s_x[];  // kInside: codes [block][token], scales [unit][half][token]
  uint8_t* s_scale = s_x + (size_t)nsb * 8 * o.M * 16;
  auto load = [&](int sb, MxStage<NMAT>& a, Tokens& b) {
    const size_t u = (size_t)sb * kMxUnit;
#pragma unroll
    for (int n = 0; n < NMAT; ++n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) a.code[n][j] = ld_stream((const i32x4*)(wp[n] + u + 1024 * j + lane * 16));
      a.scale[n] = ld_stream((const uint32_t*)(wp[n] + u + kMxCodes + lane * 4));
    }
    if constexpr (!kInside && A8) {
      const size_t u8 = (size_t)sb * kMx8Unit;
#pragma unroll
      for (int g = 0; g < MG; ++g) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int p = 0; p < 2; ++p)
            b.plane[g][j][p] = *(const i32x4*)(xp[g] + u8 + p * kMx8Plane + 1024 * j + boff[g] * 16);
        b.scale[g] = *(const uint32_t*)(xp[g] + u8 + kMx8Codes + boff[g] * 4);
      }
    } else if constexpr (!kInside) {
#pragma unroll
      for (int g = 0; g < MG; ++g) {
#pragma unroll
        for (int j = 0; j < 4; ++j) b.code[g][j] = *(const i32x4*)(xp[g] + u + 1024 * j + boff[g] * 16);
        b.scale[g] = *(const uint32_t*)(xp[g] + u + kMxCodes + boff[g] * 4);
      }
    }
  };
  // kInside: the token operands of one unit from LDS
  auto fetch = [&](int sb, MxStage<MG>& b) {
    const int tok = min(lane & 31, o.M - 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) b.code[0][j] = *(const i32x4*)(s_x + ((sb * 8 + 2 * j + half) * o.M + tok) * 16);
    b.scale[0] = *(const uint32_t*)(s_scale + ((sb * 2 + half) * o.M + tok) * 4);
  };
  f32x16 acc[NMAT][MG];
#pragma unroll
  for (int n = 0; n < NMAT; ++n)
#pragma unroll
    for (int g = 0; g < MG; ++g) acc[n][g] = f32x16{};
  auto step8 = [&](auto jc, const MxStage<NMAT>& a, const Tokens& b) {
    constexpr int J = decltype(jc)::value;
    if constexpr (A8) {
#pragma unroll
      for (int g = 0; g < MG; ++g) {
        i32x8 low = {}, high = {};
        mx8_digits(b.plane[g][J][0], 0, low, high);
        mx8_digits(b.plane[g][J][1], 1, low, high);
#pragma unroll
        for (int n = 0; n < NMAT; ++n)
          acc[n][g] = mx8_digit_product<J>(a.code[n][J], high, acc[n][g], a.scale[n], b.scale[g] + kMx8HighDigit);
#pragma unroll
        for (int n = 0; n < NMAT; ++n)
          acc[n][g] = mx8_digit_product<J>(a.code[n][J], low, acc[n][g], a.scale[n], b.scale[g]);
      }
    }
  };
  auto multiply = [&](const MxStage<NMAT>& a, const Tokens& b) {
    if constexpr (A8) {
      step8(std::integral_constant<int, 0>{}, a, b);
      step8(std::integral_constant<int, 1>{}, a, b);
      step8(std::integral_constant<int, 2>{}, a, b);
      step8(std::integral_constant<int, 3>{}, a, b);
    } else
#pragma unroll
    for (int n = 0; n < NMAT; ++n)
#pragma unroll
      for (int g = 0; g < MG; ++g) {
        acc[n][g] = mx_product<0>(a.code[n][0], b.code[g][0], acc[n][g], a.scale[n], b.scale[g]);
        acc[n][g] = mx_product<1>(a.code[n][1], b.code[g][1], acc[n][g], a.scale[n], b.scale[g]);
        acc[n][g] = mx_product<2>(a.code[n][2], b.code[g][2], acc[n][g], a.scale[n], b.scale[g]);
        acc[n][g] = mx_product<3>(a.code[n][3], b.code[g][3], acc[n][g], a.scale[n], b.scale[g]);
      }
  };
  MxStage<NMAT> a[D];
  Tokens b[kInside ? 1 : D];
  // kInside: the token rows are requested before the first weights and quantised, kXAhead chunks of 8
  // values a thread at a time, while those are on their way.  Every lane takes part in each chunk (four
  // lanes share a block); a row has nch chunks, those behind K are the padding.
  constexpr int kXAhead = 4, kXT = kInside ? XT : 0;
  MxWords<kXT> chunk[kXAhead];
  const int nch = nsb * 32, items = nch * o.M;
  auto x_row = [&](int item) {  // item / nch, for up to kMxInside rows
    int r = 0;
#pragma unroll
    for (int k = 1; k < kMxInside; ++k) r += item >= k * nch;
    return r;
  };
  auto x_load = [&](int first) {
#pragma unroll
    for (int i = 0; i < kXAhead; ++i) {
      const int item = first + i * WAVES * 64 + (int)threadIdx.x, row = x_row(item), k = (item - row * nch) * 8;
      chunk[i] = item < items && k < K ? mx_load8<kXT>(x + (size_t)row * row_bytes + (size_t)k * (XT == 2 ? 4 : 2))
                                       : MxWords<kXT>{};
    }
  };
  auto x_quantise = [&](int first) {
#pragma unroll
    for (int i = 0; i < kXAhead; ++i) {
      const int item = first + i * WAVES * 64 + (int)threadIdx.x, row = x_row(item), c = item - row * nch, kb = c >> 2;
      float f[8];
      mx_floats<kXT>(chunk[i], f);
      const uint32_t s = mx_scale_byte(max4(abs_max8(f)));
      const uint32_t code = mx_codes8(f, s);
      if (item >= items) continue;
      *(uint32_t*)(s_x + (kb * o.M + row) * 16 + (c & 3) * 4) = code;
      if ((c & 3) == 0) s_scale[(((kb >> 3) * 2 + (kb & 1)) * o.M + row) * 4 + ((kb >> 1) & 3)] = (uint8_t)s;
    }
  };
  if constexpr (kInside) x_load(0);
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (wave + d * WAVES < nsb) load(wave + d * WAVES, a[d], b[kInside ? 0 : d]);
  if constexpr (kInside) {
    x_quantise(0);
    for (int first = kXAhead * WAVES * 64; first < items; first += kXAhead * WAVES * 64) {
      x_load(first);
      x_quantise(first);
    }
    __syncthreads();
  }
  for (int sb = wave; sb < nsb; sb += D * WAVES) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int at = sb + d * WAVES;
      if (at >= nsb) break;
      if constexpr (kInside) fetch(at, b[0]);
      multiply(a[d], b[kInside ? 0 : d]);
      if (at + D * WAVES < nsb) load(at + D * WAVES, a[d], b[kInside ? 0 : d]);
    }
  }
  // lane: token lane % 32, features 8 q + 4 (lane / 32) + i; the upper half of the waves first
  float* mine = &s_part[0][0][wave % kHalfWaves][(lane & 31) * kRow + 4 * half];
  constexpr int kNext = kHalfWaves * 32 * kRow;  // from one (matrix, group) to the next
#pragma unroll
  for (int r = 1; r >= 0; --r) {
    if (wave / kHalfWaves == r) {
#pragma unroll
      for (int n = 0; n < NMAT; ++n)
#pragma unroll
        for (int g = 0; g < MG; ++g)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            f32x4* p = (f32x4*)(mine + (n * MG + g) * kNext + 8 * q);
            const f32x4 v = f32x4{acc[n][g][4 * q], acc[n][g][4 * q + 1], acc[n][g][4 * q + 2], acc[n][g][4 * q + 3]};
            *p = r ? v : *p + v;
          }
    }
    __syncthreads();
  }
  for (int item = threadIdx.x; item < MG * 256; item += WAVES * 64) {
    const int g = item >> 8, t = (item >> 3) & 31, f = (item & 7) * 4, tt = tt0 + g;
    f32x4 sum[NMAT];
#pragma unroll
    for (int n = 0; n < NMAT; ++n) {
      sum[n] = *(const f32x4*)&s_part[n][g][0][t * kRow + f];
#pragma unroll
      for (int w = 1; w < kHalfWaves; ++w) sum[n] += *(const f32x4*)&s_part[n][g][w][t * kRow + f];
    }
    mx_finish4<NMAT, MODE, A8>(o, tt, t, ft * 32 + f, item, sum);
  }
}

template <int NMAT, int WAVES, int MG, int D, int MODE, int XT, bool A8>
static int launch_stream(const MxProduct& p, hipStream_t s) {
  const dim3 grid(mx_row_tiles(p.o.N), (mx_row_tiles(p.o.M) + MG - 1) / MG);
  const int nsb = mx_ksb(p.K);
  const size_t lds = XT == kMxPackedX ? 0 : (size_t)nsb * p.o.M * (8 * 16 + 8);
  auto kern = mx_stream_kernel<NMAT, WAVES, MG, D, MODE, XT, A8>;
  launch_timed(p.slot, kern, grid, dim3(WAVES * 64), lds, s, p.x, p.w0, p.w1, nsb, p.o, p.K, p.row_bytes);
  return check_launch("mx_stream_kernel");
}

template <int MODE, int XT, bool A8>
static int launch_mode(const MxProduct& p, const MxPlan& pl, hipStream_t s) {
  constexpr int NMAT = MODE == kMxRowsOut ? 1 : 2;
  if constexpr (XT == kMxPackedX && !(A8 && NMAT == 2)) {
    if (pl.kind == kMxStreamWide) return launch_stream<NMAT, NMAT == 1 ? 8 : 4, 2, A8 ? 1 : 2, MODE, XT, A8>(p, s);
  }
  if constexpr (NMAT == 1) {
    if (pl.kind == kMxStreamDeep) return launch_stream<1, 4, 1, 2, MODE, XT, A8>(p, s);
  }
  if (pl.kind == kMxStreamLong) return launch_stream<NMAT, 8, 1, A8 ? 1 : 2, MODE, XT, A8>(p, s);
  return launch_stream<NMAT, 4, 1, 1, MODE, XT, A8>(p, s);
}

template <int MODE>
static int launch_few(const MxProduct& p, const MxPlan& pl, hipStream_t s) {
  if (p.x_type == 0) return launch_mode<MODE, 0, false>(p, pl, s);
  if (p.x_type == 1) return launch_mode<MODE, 1, false>(p, pl, s);
  if (p.x_type == 2) return launch_mode<MODE, 2, false>(p, pl, s);
  return launch_mode<MODE, kMxPackedX, false>(p, pl, s);
}

int launch_mx_stream(const MxProduct& p, const MxPlan& pl, hipStream_t s) {
  if (p.a8) {
    if (p.mode == kMxRowsOut) return launch_mode<kMxRowsOut, kMxPackedX, true>(p, pl, s);
    if (p.mode == kMxGated) return launch_mode<kMxGated, kMxPackedX, true>(p, pl, s);
    return launch_mode<kMxPacked8, kMxPackedX, true>(p, pl, s);
  }
  if (p.mode == kMxRowsOut) return launch_few<kMxRowsOut>(p, pl, s);
  if (p.mode == kMxGated) return launch_few<kMxGated>(p, pl, s);
  return launch_few<kMxPacked>(p, pl, s);
}

}  // namespace qmlp
