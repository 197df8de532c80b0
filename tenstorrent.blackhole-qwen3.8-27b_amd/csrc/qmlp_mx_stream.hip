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
#include "qmlp_internal.h"
#include "qmlp_mx.h"

namespace qmlp {

// One 256-K unit of N 32-row matrices: the lane's 16 code bytes of the four K-steps and the dword with
// their scales.
template <int N>
struct MxStage {
  i32x4 code[N][4];
  uint32_t scale[N];
};

// out^T[features, tokens] = W x^T: the weights as the A operand, MG groups of 32 token rows as B.  The
// waves of a workgroup share the units of K out in turn, so that it reads every weight matrix front to
// back, and add their sums up in a fixed order through LDS (deterministic).
template <int NMAT, int WAVES, int MG, int D, int MODE, int XT>
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
    xp[g] = x + (size_t)tt * nsb * kMxUnit;
    boff[g] = half * 32 + min(lane & 31, o.M - 1 - tt * 32);
  }
  constexpr bool kInside = XT != kMxPackedX;
  extern __shared__ __align__(16) uint8_t s_x[];  // kInside: codes [block][token], scales [unit][half][token]
  uint8_t* s_scale = s_x + (size_t)nsb * 8 * o.M * 16;
  auto load = [&](int sb, MxStage<NMAT>& a, MxStage<MG>& b) {
    const size_t u = (size_t)sb * kMxUnit;
#pragma unroll
    for (int n = 0; n < NMAT; ++n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) a.code[n][j] = ld_stream((const i32x4*)(wp[n] + u + 1024 * j + lane * 16));
      a.scale[n] = ld_stream((const uint32_t*)(wp[n] + u + kMxCodes + lane * 4));
    }
    if constexpr (!kInside) {
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
  auto multiply = [&](const MxStage<NMAT>& a, const MxStage<MG>& b) {
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
  MxStage<MG> b[kInside ? 1 : D];
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
    const int m = tt * 32 + t, n0 = ft * 32 + f;
    if constexpr (MODE == kMxRowsOut) {
      mx_store4(o, m, n0, sum[0]);
    } else {
      f32x4 h;
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = silu_mul(sum[0][i], sum[NMAT - 1][i]);
      if constexpr (MODE == kMxGated) {
        mx_store4(o, m, n0, h);
      } else {  // the 32 features of a token are one block, in 8 neighbouring lanes
        uint32_t mx = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = max(mx, __float_as_uint(h[i]) & 0x7fffffffu);
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, d));
        const uint32_t s = mx_scale_byte(mx);
        const uint32_t c = mx_codes4(h, s);
        const uint32_t hi = (uint32_t)__shfl_xor((int)c, 1);
        if (m < o.M) {
          uint8_t* unit = (uint8_t*)o.out + ((size_t)tt * mx_ksb(o.N) + n0 / kMxK) * kMxUnit;
          const int kb = (n0 % kMxK) / kMxBlock;
          if ((item & 1) == 0) *(uint32_t*)(unit + (kb * 32 + t) * 16 + f / 2) = c | (hi << 16);
          if ((item & 7) == 0) unit[kMxCodes + 4 * (t + 32 * (kb & 1)) + (kb >> 1)] = (uint8_t)s;
        }
      }
    }
  }
}

template <int NMAT, int WAVES, int MG, int D, int MODE, int XT>
static int launch_stream(const MxProduct& p, hipStream_t s) {
  const dim3 grid(mx_row_tiles(p.o.N), (mx_row_tiles(p.o.M) + MG - 1) / MG);
  const int nsb = mx_ksb(p.K);
  const size_t lds = XT == kMxPackedX ? 0 : (size_t)nsb * p.o.M * (8 * 16 + 8);
  launch_timed(p.slot, mx_stream_kernel<NMAT, WAVES, MG, D, MODE, XT>, grid, dim3(WAVES * 64), lds, s, p.x, p.w0, p.w1,
               nsb, p.o, p.K, p.row_bytes);
  return check_launch("mx_stream_kernel");
}

template <int MODE, int XT>
static int launch_mode(const MxProduct& p, const MxPlan& pl, hipStream_t s) {
  constexpr int NMAT = MODE == kMxRowsOut ? 1 : 2;
  if constexpr (XT == kMxPackedX) {
    if (pl.kind == kMxStreamWide) return launch_stream<NMAT, NMAT == 1 ? 8 : 4, 2, 2, MODE, XT>(p, s);
  }
  if constexpr (NMAT == 1) {
    if (pl.kind == kMxStreamDeep) return launch_stream<1, 4, 1, 2, MODE, XT>(p, s);
  }
  if (pl.kind == kMxStreamLong) return launch_stream<NMAT, 8, 1, 2, MODE, XT>(p, s);
  return launch_stream<NMAT, 4, 1, 1, MODE, XT>(p, s);
}

template <int MODE>
static int launch_few(const MxProduct& p, const MxPlan& pl, hipStream_t s) {
  if (p.x_type == 0) return launch_mode<MODE, 0>(p, pl, s);
  if (p.x_type == 1) return launch_mode<MODE, 1>(p, pl, s);
  if (p.x_type == 2) return launch_mode<MODE, 2>(p, pl, s);
  return launch_mode<MODE, kMxPackedX>(p, pl, s);
}

int launch_mx_stream(const MxProduct& p, const MxPlan& pl, hipStream_t s) {
  if (p.mode == kMxRowsOut) return launch_few<kMxRowsOut>(p, pl, s);
  if (p.mode == kMxGated) return launch_few<kMxGated>(p, pl, s);
  return launch_few<kMxPacked>(p, pl, s);
}

}  // namespace qmlp
