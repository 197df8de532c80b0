// qmlp_mx_stream.hip -- MXFP4 products: packed weights times packed activations, one workgroup per 32
// features x 32 tokens (layout: qmlp_mx.h).
#include "qmlp_internal.h"
#include "qmlp_mx.h"

namespace qmlp {

// One 256-K unit of every operand of a wave: the lane's 16 code bytes of the four K-steps, and the
// dword with their scales.
template <int N>
struct MxStage {
  i32x4 code[N][4];
  uint32_t scale[N];
};

// out^T[features, tokens] = W x^T: the weights as the A operand, 32 token rows as B.  The waves of a
// workgroup share the units of K out in turn, so that it reads every weight matrix front to back, and
// add their sums up in wave order through LDS (deterministic).
template <int NMAT, int WAVES, int MODE>
__global__ __launch_bounds__(WAVES * 64) void mx_stream_kernel(const uint8_t* __restrict__ x,
                                                              const uint8_t* __restrict__ w0,
                                                              const uint8_t* __restrict__ w1, int nsb, MxOut o) {
  constexpr int kRow = 36;  // floats a token's 32 features take in LDS
  __shared__ float s_part[NMAT][WAVES][32 * kRow];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ft = blockIdx.x, tt = blockIdx.y;
  const int trow = min(lane & 31, o.M - 1 - tt * 32), half = lane >> 5;
  const uint8_t* wp[2] = {w0 + (size_t)ft * nsb * kMxUnit, NMAT > 1 ? w1 + (size_t)ft * nsb * kMxUnit : nullptr};
  const uint8_t* xp = x + (size_t)tt * nsb * kMxUnit;
  const uint32_t aoff = lane * 16, soff = kMxCodes + lane * 4;
  const uint32_t boff = (half * 32 + trow) * 16, tsoff = kMxCodes + (half * 32 + trow) * 4;

  auto load = [&](int sb, MxStage<NMAT>& a, MxStage<1>& b) {
    const size_t u = (size_t)sb * kMxUnit;
#pragma unroll
    for (int j = 0; j < 4; ++j) b.code[0][j] = *(const i32x4*)(xp + u + boff + 1024 * j);
    b.scale[0] = *(const uint32_t*)(xp + u + tsoff);
#pragma unroll
    for (int n = 0; n < NMAT; ++n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) a.code[n][j] = ld_stream((const i32x4*)(wp[n] + u + aoff + 1024 * j));
      a.scale[n] = ld_stream((const uint32_t*)(wp[n] + u + soff));
    }
  };
  f32x16 acc[NMAT];
#pragma unroll
  for (int n = 0; n < NMAT; ++n) acc[n] = f32x16{};
  auto multiply = [&](const MxStage<NMAT>& a, const MxStage<1>& b) {
#pragma unroll
    for (int n = 0; n < NMAT; ++n) {
      acc[n] = mx_product<0>(a.code[n][0], b.code[0][0], acc[n], a.scale[n], b.scale[0]);
      acc[n] = mx_product<1>(a.code[n][1], b.code[0][1], acc[n], a.scale[n], b.scale[0]);
      acc[n] = mx_product<2>(a.code[n][2], b.code[0][2], acc[n], a.scale[n], b.scale[0]);
      acc[n] = mx_product<3>(a.code[n][3], b.code[0][3], acc[n], a.scale[n], b.scale[0]);
    }
  };
  for (int sb = wave; sb < nsb; sb += WAVES) {
    MxStage<NMAT> a;
    MxStage<1> b;
    load(sb, a, b);
    multiply(a, b);
  }
  // lane: token lane % 32, features 8 (i / 4) + 4 (lane / 32) + i % 4
#pragma unroll
  for (int n = 0; n < NMAT; ++n)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *(f32x4*)&s_part[n][wave][(lane & 31) * kRow + 8 * q + 4 * half] =
          f32x4{acc[n][4 * q], acc[n][4 * q + 1], acc[n][4 * q + 2], acc[n][4 * q + 3]};
  __syncthreads();
  if (threadIdx.x >= 256) return;
  const int t = threadIdx.x >> 3, f = (threadIdx.x & 7) * 4;
  f32x4 sum[NMAT];
#pragma unroll
  for (int n = 0; n < NMAT; ++n) {
    sum[n] = *(const f32x4*)&s_part[n][0][t * kRow + f];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum[n] += *(const f32x4*)&s_part[n][w][t * kRow + f];
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
        if ((threadIdx.x & 1) == 0) *(uint32_t*)(unit + (kb * 32 + t) * 16 + f / 2) = c | (hi << 16);
        if ((threadIdx.x & 7) == 0) unit[kMxCodes + 4 * (t + 32 * (kb & 1)) + (kb >> 1)] = (uint8_t)s;
      }
    }
  }
}

template <int NMAT, int MODE>
static int launch(const MxProduct& p, hipStream_t s) {
  const dim3 grid(mx_row_tiles(p.o.N), mx_row_tiles(p.o.M));
  launch_timed(p.slot, mx_stream_kernel<NMAT, 4, MODE>, grid, dim3(256), 0, s, p.x, p.w0, p.w1, mx_ksb(p.K), p.o);
  return check_launch("mx_stream_kernel");
}

int launch_mx_product(const MxProduct& p, hipStream_t s) {
  if (p.mode == kMxRowsOut) return launch<1, kMxRowsOut>(p, s);
  if (p.mode == kMxGated) return launch<2, kMxGated>(p, s);
  return launch<2, kMxPacked>(p, s);
}

}  // namespace qmlp
