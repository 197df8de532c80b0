// qmlp_mx8_few.hip -- products of up to 16 tokens in MXINT8 with MXFP4 weights: one workgroup per 32 features
// (layouts: qmlp_mx.h, qmlp_mx8.h).
//
// Bound by the weights, as the streamed products of 4-bit activations are (qmlp_mx_stream.hip).  Here the 16x16x128
// scaled product is the one to take: its token operand is 16 rows of four blocks, where the 32x32x64 product's is 32
// rows of two, so that up to 16 tokens cost half the loads, half the digits and half the products.
//
// Measured with four sets of weights in turn: one token of 17408 -> 5120 12.2-13.1 us (3.6-3.9 TB/s; 160 workgroups,
// one to a CU, each of which quantises the token), 16 tokens of the pair 5120 -> 17408 20.6-21.2 (4.5 TB/s).
#include <type_traits>

#include "qmlp_internal.h"
#include "qmlp_mx8.h"

namespace qmlp {

// A lane: row lane % 16 of each half of a 32-row weight unit, block 4 j + lane / 16 of K-step j (128 K).
template <int NMAT>
struct Mx8FewWeights {
  i32x4 code[NMAT][2][2];  // [half][K-step]
  uint32_t scale[NMAT][2];  // byte 2 j: K-step j's
};
struct Mx8FewTokens {
  i32x4 plane[2][2];  // [K-step][plane]
  uint32_t scale;
};

template <int J>
__device__ __forceinline__ f32x4 mx8_few_product(i32x4 a, const i32x8& digit, f32x4 c, uint32_t sa, uint32_t sb) {
  const i32x8 a8 = __builtin_shufflevector(a, i32x4{0, 0, 0, 0}, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, digit, c, 4, 2, 2 * J, (int)sa, 2 * J, (int)sb);
}

// The waves of a workgroup share the units of K out in turn and add their sums up in a fixed order through LDS
// (deterministic).  XT: type of unpacked rows that the workgroup quantises by itself, or kMxPackedX.
template <int NMAT, int WAVES, int MODE, int XT>
__global__ __launch_bounds__(WAVES * 64) void mx8_few_kernel(const uint8_t* __restrict__ x,
                                                            const uint8_t* __restrict__ w0,
                                                            const uint8_t* __restrict__ w1, int nsb, MxOut o, int K,
                                                            size_t row_bytes) {
  constexpr int kRow = 36;  // floats a token's 32 features take in LDS
  constexpr int kHalfWaves = WAVES / 2;
  constexpr bool kInside = XT != kMxPackedX;
  __shared__ float s_part[NMAT][kHalfWaves][16 * kRow];
  extern __shared__ __align__(16) uint8_t s_x[];  // kInside: groups [block][token][2], scales [unit][half][token]
  uint8_t* s_scale = s_x + (size_t)nsb * 8 * o.M * 32;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ft = blockIdx.x, g = lane >> 4, r = lane & 15, shift = 8 * (g >> 1);
  const uint8_t* wp[2] = {w0 + (size_t)ft * nsb * kMxUnit, NMAT > 1 ? w1 + (size_t)ft * nsb * kMxUnit : nullptr};
  const bool token = r < o.M;
  auto load = [&](int sb, Mx8FewWeights<NMAT>& a, Mx8FewTokens& b) {
    const size_t u = (size_t)sb * kMxUnit, u8 = (size_t)sb * kMx8Unit;
#pragma unroll
    for (int n = 0; n < NMAT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          a.code[n][h][j] = ld_stream((const i32x4*)(wp[n] + u + 2048 * j + 512 * g + 256 * h + 16 * r));
        a.scale[n][h] = ld_stream((const uint32_t*)(wp[n] + u + kMxCodes + 4 * (r + 16 * h + 32 * (g & 1))));
      }
    if constexpr (!kInside) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int p = 0; p < 2; ++p)
          b.plane[j][p] = token ? *(const i32x4*)(x + u8 + p * kMx8Plane + (2 * j + (g >> 1)) * 1024 +
                                                  (r + 32 * (g & 1)) * 16)
                                : i32x4{0, 0, 0, 0};
      b.scale = token ? *(const uint32_t*)(x + u8 + kMx8Codes + 4 * (r + 32 * (g & 1))) : 0x7f7f7f7fu;
    }
  };
  auto fetch = [&](int sb, Mx8FewTokens& b) {  // kInside
    const int tok = min(r, o.M - 1);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int p = 0; p < 2; ++p)
        b.plane[j][p] = *(const i32x4*)(s_x + ((sb * 8 + 4 * j + g) * o.M + tok) * 32 + 16 * p);
    b.scale = *(const uint32_t*)(s_scale + ((sb * 2 + (g & 1)) * o.M + tok) * 4);
  };
  f32x4 acc[NMAT][2];
#pragma unroll
  for (int n = 0; n < NMAT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) acc[n][h] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto step = [&](auto jc, const Mx8FewWeights<NMAT>& a, const Mx8FewTokens& b) {
    constexpr int J = decltype(jc)::value;
    i32x8 low = {}, high = {};
    mx8_digits(b.plane[J][0], 0, low, high);
    mx8_digits(b.plane[J][1], 1, low, high);
    const uint32_t sl = b.scale >> shift, sh = (b.scale + kMx8HighDigit) >> shift;
#pragma unroll
    for (int n = 0; n < NMAT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        acc[n][h] = mx8_few_product<J>(a.code[n][h][J], high, acc[n][h], a.scale[n][h] >> shift, sh);
#pragma unroll
    for (int n = 0; n < NMAT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        acc[n][h] = mx8_few_product<J>(a.code[n][h][J], low, acc[n][h], a.scale[n][h] >> shift, sl);
  };
  Mx8FewWeights<NMAT> a;
  Mx8FewTokens b;
  // kInside: the token rows are requested before the first weights and quantised, kXAhead chunks of 16 values a
  // thread at a time, while those are on their way.  Every lane takes part in each chunk (two lanes share a
  // block); a row has nch chunks, those behind K are the padding.
  constexpr int kXAhead = 2, kXT = kInside ? XT : 0;
  MxWords<kXT> chunk[kXAhead][2];
  const int nch = nsb * 16, items = nch * o.M;
  auto x_row = [&](int item) {  // item / nch, for up to kMxInside rows
    int row = 0;
#pragma unroll
    for (int k = 1; k < kMxInside; ++k) row += item >= k * nch;
    return row;
  };
  auto x_load = [&](int first) {
#pragma unroll
    for (int i = 0; i < kXAhead; ++i) {
      const int item = first + i * WAVES * 64 + (int)threadIdx.x, row = x_row(item), k = (item - row * nch) * 16;
      if (item < items && k < K)
        mx8_load<kXT>(x + (size_t)row * row_bytes + (size_t)k * (XT == 2 ? 4 : 2), chunk[i]);
      else
        chunk[i][0] = chunk[i][1] = MxWords<kXT>{};
    }
  };
  auto x_quantise = [&](int first) {
#pragma unroll
    for (int i = 0; i < kXAhead; ++i) {
      const int item = first + i * WAVES * 64 + (int)threadIdx.x, row = x_row(item), c = item - row * nch, kb = c >> 1;
      float f[16];
      mx8_floats<kXT>(chunk[i], f);
      uint32_t top = abs_max16(f);
      top = max(top, (uint32_t)__shfl_xor((int)top, 1));
      const uint32_t s = mx8_scale_byte(top);
      const i32x4 group = mx8_group(f, s);
      if (item >= items) continue;
      *(i32x4*)(s_x + (kb * o.M + row) * 32 + (c & 1) * 16) = group;
      if ((c & 1) == 0) s_scale[(((kb >> 3) * 2 + (kb & 1)) * o.M + row) * 4 + ((kb >> 1) & 3)] = (uint8_t)s;
    }
  };
  if constexpr (kInside) x_load(0);
  if (wave < nsb) load(wave, a, b);
  if constexpr (kInside) {
    x_quantise(0);
    for (int first = kXAhead * WAVES * 64; first < items; first += kXAhead * WAVES * 64) {
      x_load(first);
      x_quantise(first);
    }
    __syncthreads();
  }
  for (int sb = wave; sb < nsb; sb += WAVES) {
    if constexpr (kInside) fetch(sb, b);
    step(std::integral_constant<int, 0>{}, a, b);
    step(std::integral_constant<int, 1>{}, a, b);
    if (sb + WAVES < nsb) load(sb + WAVES, a, b);
  }
  // lane: token lane % 16, features 16 h + 4 (lane / 16) + i; the upper half of the waves first
  float* mine = &s_part[0][wave % kHalfWaves][r * kRow + 4 * g];
#pragma unroll
  for (int q = 1; q >= 0; --q) {
    if (wave / kHalfWaves == q) {
#pragma unroll
      for (int n = 0; n < NMAT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f32x4* p = (f32x4*)(mine + n * (kHalfWaves * 16 * kRow) + 16 * h);
          *p = q ? acc[n][h] : *p + acc[n][h];
        }
    }
    __syncthreads();
  }
  for (int item = threadIdx.x; item < 128; item += WAVES * 64) {
    const int t = item >> 3, f = (item & 7) * 4;
    f32x4 sum[NMAT];
#pragma unroll
    for (int n = 0; n < NMAT; ++n) {
      sum[n] = *(const f32x4*)&s_part[n][0][t * kRow + f];
#pragma unroll
      for (int w = 1; w < kHalfWaves; ++w) sum[n] += *(const f32x4*)&s_part[n][w][t * kRow + f];
    }
    mx_finish4<NMAT, MODE, true>(o, 0, t, ft * 32 + f, item, sum);
  }
}

template <int NMAT, int WAVES, int MODE, int XT>
static int launch_kernel(const MxProduct& p, hipStream_t s) {
  const int nsb = mx_ksb(p.K);
  const size_t lds = XT == kMxPackedX ? 0 : (size_t)nsb * p.o.M * (8 * 32 + 8);
  auto kern = mx8_few_kernel<NMAT, WAVES, MODE, XT>;
  launch_timed(p.slot, kern, dim3(mx_row_tiles(p.o.N)), dim3(WAVES * 64), lds, s, p.x, p.w0, p.w1, nsb, p.o, p.K,
               p.row_bytes);
  return check_launch("mx8_few_kernel");
}

template <int MODE, int XT>
static int launch_plan(const MxProduct& p, const MxPlan& pl, hipStream_t s) {
  constexpr int NMAT = MODE == kMxRowsOut ? 1 : 2;
  // One unit under way a wave: two take registers that cost resident workgroups (17408 x 5120 at 16 tokens, us: 13.7
  // with one, 16.0 with two; two such matrices 21.0 and 25.6).  Where every CU has workgroups enough, four waves
  // quantise their rows sooner than eight (one token of 17408 x 5120: 11.8 and 14.2, two matrices 20.1 and 25.5; of
  // 5120 x 17408, fewer workgroups than CUs, 18.7 and 14.3).
  if constexpr (XT != kMxPackedX) {
    if (pl.height == 4) return launch_kernel<NMAT, 4, MODE, XT>(p, s);
  }
  return launch_kernel<NMAT, 8, MODE, XT>(p, s);
}

template <int MODE>
static int launch_mode(const MxProduct& p, const MxPlan& pl, hipStream_t s) {
  if (p.x_type == 0) return launch_plan<MODE, 0>(p, pl, s);
  if (p.x_type == 1) return launch_plan<MODE, 1>(p, pl, s);
  if (p.x_type == 2) return launch_plan<MODE, 2>(p, pl, s);
  return launch_plan<MODE, kMxPackedX>(p, pl, s);
}

int launch_mx8_few(const MxProduct& p, const MxPlan& pl, hipStream_t s) {
  if (p.mode == kMxRowsOut) return launch_mode<kMxRowsOut>(p, pl, s);
  if (p.mode == kMxGated) return launch_mode<kMxGated>(p, pl, s);
  return launch_mode<kMxPacked8>(p, pl, s);
}

}  // namespace qmlp
