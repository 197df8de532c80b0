// qmlp_mx_tiled.hip -- MXFP4 products of many tokens (layout: qmlp_mx.h).
//
// out^T[features, tokens] = W x^T in 256 features (128 of gate and of up) x 64, 128, 192 or 256 tokens a
// workgroup of 8 waves, on the scaled 32x32x64 product, which takes codes and scale bytes as they lie in
// memory: 32 cycles for 131072 flop, 10 PFLOP/s at 2.4 GHz.  Per K unit a 256 x 256 tile reads 69.6 KB
// and multiplies for 2048 cycles of each SIMD, so what costs is moving operands about:
//   * memory -> LDS by loads that bypass the registers: the packed layout is the products' operand
//     order, so a unit comes in as it lies, and LDS is read lane by lane (no conflicts, no swizzle);
//   * LDS holds four halves (128 K) of a K unit, so that a load has two of them, 2000 cycles and more,
//     to arrive; one workgroup takes a CU;
//   * the operands of a K-step are read while the products of the one before run, one or two reads to a
//     pair of products, in the order written here.
// Measured (256 tiles of 256 x 256, K = 17408, random codes): 126-131 us, 4.5-4.6 PFLOP/s; without the
// loads into LDS 110-130, without the LDS reads 105-120, without both 94-104, while the clock goes from
// 1.70 to 1.81, 1.93 and 2.12 GHz at 64-70 % busy matrix cores: power takes its part through the clock,
// which falls as more data moves.  What idles the matrix cores a third of the cycles, in all four alike, is
// not known.  Products from registers alone reach 6.1-6.5 PFLOP/s on random codes (8.1-8.8 on constant
// ones).  Four waves of 128 x 128, which read a third less from LDS, took 127-129 us.
#include <atomic>
#include <type_traits>

#include "../../include/qwen_mlp.h"
#include "qmlp_internal.h"
#include "qmlp_mx8.h"
#include "qmlp_xcd.h"

namespace qmlp {

// 16 (or 4) bytes a lane straight from memory into LDS: lane l's, from off + its lane_off of the
// buffer, go to lds + 16 l (4 l).  off and lds are uniform.  (The host pass knows only the sizes of older
// GPUs and would drop the kernel without a word.)
typedef __attribute__((address_space(3))) void LdsVoid;
__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t src, uint32_t lane_off, int off, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (LdsVoid*)(uintptr_t)lds, 16, lane_off, off, 0, 0);
#endif
}
__device__ __forceinline__ void load_lds4(__amdgpu_buffer_rsrc_t src, uint32_t lane_off, int off, uint32_t lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (LdsVoid*)(uintptr_t)lds, 4, lane_off, off, 0, 0);
#endif
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// Waits until at most N of this wave's loads into LDS are still under way and its LDS reads are done,
// then for the workgroup.  (__syncthreads would wait for all of the loads.)
template <int N>
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(N) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The lanes of a wave see each other's LDS accesses in program order; this keeps the compiler to it.
__device__ __forceinline__ void turn_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Finishes 32 features x 32 tokens from the matrices' sums as the product leaves them: lane: token lane %
// 32, v[.][k][i]: feature 8 k + 4 (lane / 32) + i.  Rows go through `turn`, kMxTurn floats of LDS that
// belong to the wave, so that 8 lanes write 32 features of a token together: 2048 x 17408 x 512 took
// 24.5 us; written as the product leaves them, 16 bytes here and there, 34.6.
constexpr int kMxTurnRow = 36;  // floats of a token's row: 8 lanes' 16-byte accesses meet no bank twice
constexpr int kMxTurn = 32 * kMxTurnRow;
template <int NMAT, int MODE, bool A8>
__device__ __forceinline__ void mx_finish(const MxOut& o, int tok_unit, int feat_unit, int lane, float* turn,
                                          f32x4 (&v)[NMAT][4]) {
  const int half = lane >> 5, row = lane & 31, m = tok_unit * 32 + row;
  if constexpr (A8 && MODE != kMxRowsOut) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[0][k] += mx_addend(o.gate_add, o, m, feat_unit * 32 + 8 * k + 4 * half);
      v[NMAT - 1][k] += mx_addend(o.up_add, o, m, feat_unit * 32 + 8 * k + 4 * half);
    }
  }
  f32x4 y[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) y[k][i] = MODE == kMxRowsOut ? v[0][k][i] : silu_mul(v[0][k][i], v[NMAT - 1][k][i]);
  if constexpr (MODE == kMxRowsOut || MODE == kMxGated) {
#pragma unroll
    for (int k = 0; k < 4; ++k) *(f32x4*)(turn + row * kMxTurnRow + 8 * k + 4 * half) = y[k];
    turn_fence();
    const int r = lane >> 3, f = (lane & 7) * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x4 w = *(const f32x4*)(turn + (8 * k + r) * kMxTurnRow + f);
      mx_store4(o, tok_unit * 32 + 8 * k + r, feat_unit * 32 + f, w);
    }
    turn_fence();
  } else {  // a token's 32 features are one block, in lanes l and l + 32
    uint32_t mx = 0u;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = max(mx, __float_as_uint(y[k][i]) & 0x7fffffffu);
    mx = max(mx, (uint32_t)__shfl_xor((int)mx, 32));
    if constexpr (MODE == kMxPacked8) {  // each of the two lanes makes 16 neighbouring values' group
      const uint32_t s = mx8_scale_byte(mx);
      float f[16];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float mine = half ? y[2 + k][i] : y[k][i];
          const float other = __shfl_xor(half ? y[k][i] : y[2 + k][i], 32);
          f[8 * k + i] = half ? other : mine;
          f[8 * k + 4 + i] = half ? mine : other;
        }
      const i32x4 group = mx8_group(f, s);
      if (m < o.M && feat_unit * 32 < o.N) {
        uint8_t* unit = (uint8_t*)o.out + ((size_t)tok_unit * mx_ksb(o.N) + feat_unit / 8) * kMx8Unit;
        *(i32x4*)(unit + mx8_at(row, feat_unit % 8, half)) = group;
        if (half == 0) unit[mx8_scale_at(row, feat_unit % 8)] = (uint8_t)s;
      }
      return;
    }
    const uint32_t s = mx_scale_byte(mx);
    u32x4 c;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t mine = mx_codes4(y[k], s);
      c[k] = mine | ((uint32_t)__shfl_xor((int)mine, 32) << 16);  // in K order for the lower lanes
    }
    if (half == 0 && m < o.M && feat_unit * 32 < o.N) {
      uint8_t* unit = (uint8_t*)o.out + ((size_t)tok_unit * mx_ksb(o.N) + feat_unit / 8) * kMxUnit;
      const int kb = feat_unit % 8;
      *(u32x4*)(unit + (kb * 32 + row) * 16) = c;
      unit[kMxCodes + 4 * (row + 32 * (kb & 1)) + (kb >> 1)] = (uint8_t)s;
    }
  }
}

// NF x NT waves, each WF x WT products of 32 features x 32 tokens (WF: of all matrices together).  8-bit
// activations (XP = 2): a token unit's two planes are loaded and kept like two units of 4-bit codes, each with
// the scales, and a product is two, one for each digit.
template <int NMAT, int WF, int WT, int NF, int NT, int XP>
struct MxTile {
  static constexpr int kWaves = NF * NT;
  static constexpr int kFeatUnits = WF * NF;
  static constexpr int kTokUnits = WT * NT;
  static constexpr int kUnits = kFeatUnits + kTokUnits * XP;
  static constexpr int kFeatures = 32 * kFeatUnits / NMAT;
  static constexpr int kTokens = 32 * kTokUnits;
  static constexpr int kHalf = kUnits * (kMxCodes / 2);  // codes of 128 K
  static constexpr int kLds = 4 * kHalf + 2 * kUnits * 256;
  static constexpr int kMine = (kUnits + kWaves - 1) / kWaves;  // units a wave brings in
  static_assert(kLds <= 160 * 1024 && WF * WT * XP % 2 == 0, "tile");
};

template <int NMAT, int WF, int WT, int NF, int NT, int MODE, int XP>
__global__ __launch_bounds__(NF* NT * 64, 1) void mx_tiled_kernel(const uint8_t* __restrict__ x,
                                                                  const uint8_t* __restrict__ w0,
                                                                  const uint8_t* __restrict__ w1, int nsb, int ntt,
                                                                  int whole, int ks, f32x4* __restrict__ parts,
                                                                  MxOut o) {
  using T = MxTile<NMAT, WF, WT, NF, NT, XP>;
  extern __shared__ __align__(16) uint8_t s_stage[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wf = wave % NF, wt = wave / NF;
  // the tile, and the piece q of its K units: the first `whole` tiles run whole, the others in ks pieces
  const bool split = (int)blockIdx.x >= whole && ks > 1;
  const int piece = (int)blockIdx.x < whole ? xcd_run(blockIdx.x, whole) : xcd_run(blockIdx.x - whole, gridDim.x - whole);
  const int pieces = split ? ks : 1;
  const int tile = (int)blockIdx.x < whole ? piece : whole + piece / pieces, q = split ? piece % pieces : 0;
  const int ft = tile / ntt, tt = tile % ntt;
  const int u0 = q * nsb / pieces, n = (q + 1) * nsb / pieces - u0;
  const int ftiles = mx_row_tiles(o.N), ttiles = mx_row_tiles(o.M);
  const uint32_t lds0 = lds_address(s_stage);
  const uint32_t lds_scales = lds0 + 4 * T::kHalf;
  const uint32_t lane16 = lane * 16, lane4 = lane * 4;
  // The units this wave brings in.  Unit order: wave column by wave column its matrices one after the
  // other, then the tokens; units behind the last row tile repeat it (their sums are not stored).  Where
  // the units do not divide by the waves, the last one is brought in several times (the same bytes to the
  // same place), so that every wave waits for the same number of loads: 16 for 10 units at 64 tokens, 12
  // at 128, 14 at 192.
  __amdgpu_buffer_rsrc_t src[T::kMine];
  int unit_bytes[T::kMine], scales_at[T::kMine];
#pragma unroll
  for (int i = 0; i < T::kMine; ++i) {
    const int u = min(wave * T::kMine + i, T::kUnits - 1);  // the last one again where they do not divide
    const uint8_t* p;
    int extent = n * kMxUnit;
    unit_bytes[i] = kMxUnit;
    scales_at[i] = kMxCodes;
    if (u < T::kFeatUnits) {
      constexpr int per = WF / NMAT;
      const int col = u / WF, mat = (u % WF) / per, f = col * per + u % per;
      const int row = min(ft * (T::kFeatUnits / NMAT) + f, ftiles - 1);
      p = (NMAT > 1 && mat ? w1 : w0) + (size_t)row * nsb * kMxUnit;
      p += (size_t)u0 * kMxUnit;
    } else if constexpr (XP == 1) {
      p = x + ((size_t)min(tt * T::kTokUnits + u - T::kFeatUnits, ttiles - 1) * nsb + u0) * kMxUnit;
    } else {
      const int v = u - T::kFeatUnits, plane = v % XP * kMx8Plane;
      p = x + ((size_t)min(tt * T::kTokUnits + v / XP, ttiles - 1) * nsb + u0) * kMx8Unit + plane;
      unit_bytes[i] = kMx8Unit;
      scales_at[i] = kMx8Codes - plane;
      extent = n * kMx8Unit - plane;
    }
    src[i] = __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, extent, kBufferRsrcWord3);
  }
  // A half of a K unit comes in two parts, half of the wave's units each: load k of part `part` of half h
  // of unit sb.  The codes go to slot 2 (sb % 2) + h, with half 0 the unit's scales.
  constexpr int kPart0 = T::kMine / 2, kPart1 = T::kMine - kPart0;
  auto issue = [&](int sb, int h, int part, int k) {
    const int per = h == 0 ? 3 : 2, i = part * kPart0 + k / per, c = k % per;
    if (k >= per * (part ? kPart1 : kPart0)) return;
    const int u = min(wave * T::kMine + i, T::kUnits - 1);
    if (c < 2)
      load_lds16(src[i], lane16, sb * unit_bytes[i] + 2048 * h + 1024 * c,
                   lds0 + (2 * (sb & 1) + h) * T::kHalf + u * 2048 + c * 1024);
    else
      load_lds4(src[i], lane4, sb * unit_bytes[i] + scales_at[i], lds_scales + ((sb & 1) * T::kUnits + u) * 256);
  };
  auto issue_all = [&](int sb, int h, int part) {
#pragma unroll
    for (int k = 0; k < 3 * kPart1; ++k) issue(sb, h, part, k);
  };
  f32x16 acc[WF][WT];
#pragma unroll
  for (int f = 0; f < WF; ++f)
#pragma unroll
    for (int t = 0; t < WT; ++t) acc[f][t] = f32x16{};
  constexpr int kB = WT * XP;  // token operands of a K-step
  i32x4 a[2][WF], b[2][kB];
  uint32_t fs[WF], xs[WT], fs_next[WF], xs_next[WT];
  const uint8_t* sf = s_stage + wf * WF * 2048 + lane16;
  const uint8_t* sx = s_stage + (T::kFeatUnits + wt * kB) * 2048 + lane16;
  const uint8_t* sc = s_stage + 4 * T::kHalf + lane4;
  // operand k of one K-step of the wave: its first feature unit, its tokens, its other feature units
  auto fetch = [&](int sb, int h, int j, int k) {
    const uint32_t at = (2 * (sb & 1) + h) * T::kHalf + j * 1024;
    if (k >= WF + kB) return;
    if constexpr (XP == 2) {  // the tokens first: their digits take time
      if (k < kB)
        b[j][k] = *(const i32x4*)(sx + at + k * 2048);
      else
        a[j][k - kB] = *(const i32x4*)(sf + at + (k - kB) * 2048);
      return;
    }
    if (k >= 1 && k <= kB)
      b[j][k - 1] = *(const i32x4*)(sx + at + (k - 1) * 2048);
    else
      a[j][k ? k - kB : 0] = *(const i32x4*)(sf + at + (k ? k - kB : 0) * 2048);
  };
  auto fetch_scale = [&](int sb, int k) {
    const uint8_t* s = sc + (sb & 1) * T::kUnits * 256;
    if (k < WT)
      xs_next[k] = *(const uint32_t*)(s + (T::kFeatUnits + wt * kB + k * XP) * 256);
    else if (k < WF + WT)
      fs_next[k - WT] = *(const uint32_t*)(s + (wf * WF + k - WT) * 256);
  };
  // Token units of this wave that hold tokens (none where its features lie behind the last one): the
  // last tokens' tile does no product that no output needs.
  const int mine_f = (ft * (T::kFeatUnits / NMAT) + wf * (WF / NMAT)) < ftiles ? WT : 0;
  const int nv = max(0, min(mine_f, ttiles - (tt * T::kTokUnits + wt * WT)));
  // One K-step's products, in groups of two; before each group `beside(group)` asks for what comes in
  // beside them (the order is kept as written).
  constexpr int kGroups = WF * WT * XP / 2;
  // 8-bit: the digits of a K-step's token operands and of the next one's, which are made plane by plane in front
  // of the last two groups' products
  i32x8 low[2][XP == 2 ? WT : 1], high[2][XP == 2 ? WT : 1];
  auto digits = [&](int j, int plane) {
    if constexpr (XP == 2) {
#pragma unroll
      for (int t = 0; t < WT; ++t) mx8_digits(b[j][2 * t + plane], plane, low[j][t], high[j][t]);
    }
  };
  auto multiply = [&](auto jc, auto full, auto next, auto beside) {
    constexpr int J = decltype(jc)::value, j = J & 1;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      beside(g);
      if constexpr (XP == 2) {
        if (decltype(next)::value) {
          if (g == (kGroups > 2 ? kGroups - 2 : 1)) digits(1 - j, 0);
          if (g == kGroups - 1) digits(1 - j, 1);
        }
        // two products' high digits, then their low ones: none waits for the sum before it
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int i = g / 2 * 2 + k, f = i / WT, t = i % WT;
          if (decltype(full)::value || t < nv)
            acc[f][t] = mx8_digit_product<J>(a[j][f], g % 2 ? low[j][t] : high[j][t], acc[f][t], fs[f],
                                             xs[t] + (g % 2 ? 0u : kMx8HighDigit));
        }
        __builtin_amdgcn_sched_barrier(0);
        continue;
      }
#pragma unroll
      for (int k = 2 * g; k < 2 * g + 2; ++k) {
        const int f = k / WT, t = k % WT;
        if (decltype(full)::value || t < nv)
          acc[f][t] = mx_product<J>(a[J & 1][f], b[J & 1][t], acc[f][t], fs[f], xs[t]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // item k of n spread over the groups, the first ones first
  auto spread = [&](int g, int n, auto f) {
    const int per = (n + kGroups - 1) / kGroups;
#pragma unroll
    for (int k = g * per; k < (g + 1) * per; ++k)
      if (k < n) f(k);
  };
  // One K unit in four steps.  Beside the products of a step the operands of the next one come from
  // LDS and a part of a half that is 3 to 4 halves ahead from memory: half i's slot is free once the
  // barrier inside half i has shown that every wave has read its last operands.  That barrier also
  // shows that half i + 1 is in LDS; the two after it may still be under way.
  // LEFT: K units behind this one, at most 2.
  auto unit = [&](int sb, auto left, auto full) {
    constexpr int LEFT = decltype(left)::value;
    constexpr int kAhead = T::kMine * 5;  // loads of two halves, one of them with scales
#pragma unroll
    for (int t = 0; t < WT; ++t) xs[t] = xs_next[t];
#pragma unroll
    for (int f = 0; f < WF; ++f) fs[f] = fs_next[f];
    multiply(std::integral_constant<int, 0>{}, full, std::true_type{}, [&](int g) {
      spread(g, WF + kB, [&](int k) { fetch(sb, 0, 1, k); });
      if constexpr (LEFT >= 1) spread(g, 2 * kPart1, [&](int k) { issue(sb + 1, 1, 1, k); });
    });
    stage_barrier<(LEFT >= 1 ? kAhead : 0)>();
    multiply(std::integral_constant<int, 1>{}, full, std::true_type{}, [&](int g) {
      spread(g, WF + kB, [&](int k) { fetch(sb, 1, 0, k); });
      if constexpr (LEFT >= 2) spread(g, 3 * kPart0, [&](int k) { issue(sb + 2, 0, 0, k); });
    });
    multiply(std::integral_constant<int, 2>{}, full, std::true_type{}, [&](int g) {
      spread(g, WF + kB, [&](int k) { fetch(sb, 1, 1, k); });
      if constexpr (LEFT >= 2) spread(g, 3 * kPart1, [&](int k) { issue(sb + 2, 0, 1, k); });
    });
    stage_barrier<(LEFT >= 2 ? kAhead : 0)>();
    multiply(std::integral_constant<int, 3>{}, full, std::bool_constant<LEFT >= 1>{}, [&](int g) {
      if constexpr (LEFT >= 1) {
        spread(g, WF + kB, [&](int k) { fetch(sb + 1, 0, 0, k); });
        spread(g, WF + WT, [&](int k) { fetch_scale(sb + 1, k); });
      }
      if constexpr (LEFT >= 2) spread(g, 2 * kPart0, [&](int k) { issue(sb + 2, 1, 0, k); });
    });
  };
  issue_all(0, 0, 0);
  issue_all(0, 0, 1);
  issue_all(0, 1, 0);
  issue_all(0, 1, 1);
  if (n > 1) {
    issue_all(1, 0, 0);
    issue_all(1, 0, 1);
    issue_all(1, 1, 0);
    stage_barrier<T::kMine * 5 + 2 * kPart0>();
  } else {
    stage_barrier<T::kMine * 2>();
  }
#pragma unroll
  for (int k = 0; k < WF + kB; ++k) {
    fetch_scale(0, k);
    fetch(0, 0, 0, k);
  }
  digits(0, 0);
  digits(0, 1);
  auto units = [&](auto full) {
    int sb = 0;
    for (; sb + 2 < n; ++sb) unit(sb, std::integral_constant<int, 2>{}, full);
    if (sb + 1 < n) unit(sb++, std::integral_constant<int, 1>{}, full);
    unit(sb, std::integral_constant<int, 0>{}, full);
  };
  if (nv == WT)
    units(std::true_type{});
  else
    units(std::false_type{});
  constexpr int per = WF / NMAT;
  if (WT <= 2 && split) {  // the sums as the lanes hold them; mx_sum_kernel adds the pieces up
    f32x4* at = parts + ((size_t)piece * T::kWaves + wave) * (WF * WT * 4 * 64) + lane;
#pragma unroll
    for (int f = 0; f < WF; ++f)
#pragma unroll
      for (int t = 0; t < WT; ++t)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (t < nv)
            at[((f * WT + t) * 4 + k) * 64] = f32x4{acc[f][t][4 * k], acc[f][t][4 * k + 1], acc[f][t][4 * k + 2],
                                                    acc[f][t][4 * k + 3]};
    return;
  }
  static_assert(T::kLds >= T::kWaves * kMxTurn * 4);
  float* turn = (float*)s_stage + wave * kMxTurn;
  if constexpr (MODE == kMxRowsOut || MODE == kMxGated) __syncthreads();  // the stages' readers are done
#pragma unroll
  for (int t = 0; t < WT; ++t) {
    if (t >= nv) break;
#pragma unroll
    for (int f = 0; f < per; ++f) {
      f32x4 v[NMAT][4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int m = 0; m < NMAT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[m][k][i] = acc[f + m * per][t][4 * k + i];
      mx_finish<NMAT, MODE, XP == 2>(o, tt * T::kTokUnits + wt * WT + t, ft * (T::kFeatUnits / NMAT) + wf * per + f, lane,
                            turn, v);
    }
  }
}

// Adds the pieces of split tiles up, in K order (deterministic), and finishes them: one wave for 32
// features x 32 tokens.  Bound by its reads and its launch: 4.1-4.8 us for 15.7 MB of pieces (201 tokens of
// 5120 x 8704).  A launch of its own, so that every CU takes part and no block waits for another.
template <int NMAT, int WF, int WT, int NF, int NT, int MODE, int XP>
__global__ __launch_bounds__(256) void mx_sum_kernel(const f32x4* __restrict__ parts, int whole, int tiles, int ntt,
                                                     int ks, MxOut o) {
  using T = MxTile<NMAT, WF, WT, NF, NT, XP>;
  constexpr int per = WF / NMAT, kItems = T::kWaves * per * WT;
  __shared__ __align__(16) float s_turn[4][kMxTurn];
  const int lane = threadIdx.x & 63;
  const int item = blockIdx.x * 4 + (threadIdx.x >> 6), tile = whole + item / kItems, r = item % kItems;
  if (tile >= tiles) return;
  const int wave = r / (per * WT), f = r / WT % per, t = r % WT;
  const int wf = wave % NF, wt = wave / NF, ft = tile / ntt, tt = tile % ntt;
  const int tok = tt * T::kTokUnits + wt * WT + t, feat = ft * (T::kFeatUnits / NMAT) + wf * per + f;
  if (tok >= mx_row_tiles(o.M) || feat >= mx_row_tiles(o.N)) return;  // left out by the product
  f32x4 v[NMAT][4];
#pragma unroll
  for (int m = 0; m < NMAT; ++m)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[m][k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int q = 0; q < ks; ++q) {
    const f32x4* at = parts + ((size_t)((tile - whole) * ks + q) * T::kWaves + wave) * (WF * WT * 4 * 64) + lane;
#pragma unroll
    for (int m = 0; m < NMAT; ++m)
#pragma unroll
      for (int k = 0; k < 4; ++k) v[m][k] += at[(((f + m * per) * WT + t) * 4 + k) * 64];
  }
  mx_finish<NMAT, MODE, XP == 2>(o, tok, feat, lane, s_turn[threadIdx.x >> 6], v);
}

template <typename T, int NMAT, int MODE, int WF, int WT, int NF, int NT, int XP>
static int launch_sum(const MxProduct& p, int whole, int tiles, int ntt, int ks, hipStream_t s) {
  constexpr int kItems = T::kWaves * WF / NMAT * WT;
  launch_timed_part(p.slot, 2, mx_sum_kernel<NMAT, WF, WT, NF, NT, MODE, XP>, dim3(((tiles - whole) * kItems + 3) / 4),
                    dim3(256), 0, s, (const f32x4*)p.parts, whole, tiles, ntt, ks, p.o);
  return check_launch("mx_sum_kernel");
}

template <int NMAT, int WF, int WT, int NF, int NT, int MODE, int XP>
static int launch_tile(const MxProduct& p, int whole, int ks, hipStream_t s) {
  using T = MxTile<NMAT, WF, WT, NF, NT, XP>;
  auto kern = mx_tiled_kernel<NMAT, WF, WT, NF, NT, MODE, XP>;
  static std::atomic<uint64_t> raised{0};
  if (int rc = raise_lds_once((const void*)kern, T::kLds, raised)) return rc;
  const int nft = (p.o.N + T::kFeatures - 1) / T::kFeatures, ntt = (p.o.M + T::kTokens - 1) / T::kTokens;
  const int tiles = nft * ntt;
  const size_t part_bytes = (size_t)(tiles - whole) * ks * (T::kWaves * WF * WT * 4096);
  if (ks > mx_ksb(p.K) || whole < 0 || whole > tiles || (ks > 1 && (WT > 2 || part_bytes > kMxPartBytes)))  // never planned
    return set_error(QMLP_E_WORKSPACE, "mx_tiled_kernel: %d tiles in %d pieces", tiles, ks);
  launch_timed_part(p.slot, ks > 1 ? 1 : 3, kern, dim3(whole + (tiles - whole) * ks), dim3(T::kWaves * 64), T::kLds, s, p.x, p.w0, p.w1,
                    mx_ksb(p.K), ntt, whole, ks, (f32x4*)p.parts, p.o);
  if (int rc = check_launch("mx_tiled_kernel")) return rc;
  if constexpr (WT <= 2) {  // mx_plan splits no higher tile
    if (ks > 1) return launch_sum<T, NMAT, MODE, WF, WT, NF, NT, XP>(p, whole, tiles, ntt, ks, s);
  }
  return 0;
}

template <int MODE>
static int launch_height(const MxProduct& p, const MxPlan& pl, hipStream_t s) {
  constexpr int NMAT = MODE == kMxRowsOut ? 1 : 2;
  if (pl.height == 1) return launch_tile<NMAT, 2, 1, 4, 2, MODE, 1>(p, pl.whole, pl.ks, s);
  if (pl.height == 2) return launch_tile<NMAT, 2, 2, 4, 2, MODE, 1>(p, pl.whole, pl.ks, s);
  if (pl.height == 3) return launch_tile<NMAT, 2, 3, 4, 2, MODE, 1>(p, pl.whole, pl.ks, s);
  return launch_tile<NMAT, 2, 4, 4, 2, MODE, 1>(p, pl.whole, pl.ks, s);
}

// 8-bit activations: two heights, as far as LDS goes; the higher one in waves of 128 features x 32 tokens, which make
// half the digits of 64 x 64 for as many reads from LDS.  2048 tokens of 17408 -> 5120 take 177-180 us (2.03-2.06
// PFLOP/s, 65 % of what two digits' products reach from registers alone) with the matrix cores 57 % busy at 1.70 GHz,
// 777 of the pair 5120 -> 17408 151-155.  Four waves of 256 x 32, with two thirds of the vector instructions: 182 and
// 157 (52 % busy at 1.84 GHz).  Digits made a dword at a time beside six groups of products: 177 and 152.  Tiles in
// bands of eight token blocks and pieces by K, which read 289 MB from behind the L2s instead of 503: no difference.
// gate_add and up_add cost the pair's 369 us at 2048 tokens 49 (143 MB each, read in the epilogue; 5.8 TB/s), at 777 13 of 157;
// a packed output or rows take the same time.
template <int MODE>
static int launch_height8(const MxProduct& p, const MxPlan& pl, hipStream_t s) {
  constexpr int NMAT = MODE == kMxRowsOut ? 1 : 2;
  if (pl.height == 1) return launch_tile<NMAT, 2, 1, 4, 2, MODE, 2>(p, pl.whole, pl.ks, s);
  return launch_tile<NMAT, 4, 1, 2, 4, MODE, 2>(p, pl.whole, pl.ks, s);
}

int launch_mx_tiled(const MxProduct& p, const MxPlan& pl, hipStream_t s) {
  if (p.a8) {
    if (p.mode == kMxRowsOut) return launch_height8<kMxRowsOut>(p, pl, s);
    if (p.mode == kMxGated) return launch_height8<kMxGated>(p, pl, s);
    return launch_height8<kMxPacked8>(p, pl, s);
  }
  if (p.mode == kMxRowsOut) return launch_height<kMxRowsOut>(p, pl, s);
  if (p.mode == kMxGated) return launch_height<kMxGated>(p, pl, s);
  return launch_height<kMxPacked>(p, pl, s);
}

}  // namespace qmlp
