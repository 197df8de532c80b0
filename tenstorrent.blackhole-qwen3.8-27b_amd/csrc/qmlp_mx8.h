// qmlp_mx8.h -- MXINT8 activations (8-bit integers, 32 to a power-of-two scale): layout and device helpers.
//
// A block of 32 consecutive K values v with largest magnitude in [2^E, 2^(E+1)) is q 2^(E-6), q = v / 2^(E-6)
// rounded half to even, |q| <= 127 (OCP MX's 8-bit integer elements without -128; E is kept in [-120, 126],
// so the step is a normal number).  A block with an infinity or a NaN is one as a whole.
//
// How the matrix cores take it.  The scaled product of 4-bit weights with 8-bit floating-point values keeps
// about 13 bits below a block's largest product (measured: up to 2^-13 of the summed magnitudes is lost,
// where 4-bit values lose 2^-24), and it runs at half the rate anyway.  So q is multiplied as its two
// digits, q = s (16 h + l) with h in 0..7 and l in 0..15, each an e2m3 number (h / 8 and l / 8: the code of an
// e2m3 value below 2 is the integer itself) under scales 2^(E+1) and 2^(E-3): two 4-bit x 6-bit products at the
// full rate, whose terms are exact and whose sums round as the 4-bit ones do.  6300 TFLOP/s from registers,
// 3150 for both digits; 4-bit x 8-bit: 3150.
//
// Memory holds 8 bits a value, and a lane makes its two operands from them with bit masks alone.  16 values
// ("a group") are three dwords of 6-bit fields and one more:
//   field i of the 96 bits: s (bit 5), l (bits 3..0); bit 4, which an e2m3 number below 2 has clear, holds h's
//   low bit for the field that starts in the next of the three dwords, where it lies at the same bit;
//   dword 3 holds h's two high bits of every field at the bits they take in whichever dword theirs is (the
//   three dwords' places for them are disjoint and fill 32 bits).
// Units of 32 rows x 256 K, 8448 B: two planes of 4096 B (the first and the last 16 values of every block) in
// the order of a 4-bit unit (qmlp_mx.h: lane l of K-step j reads 16 bytes at 1024 j + 16 l), then the scale
// bytes E + 124 (the low digit's scale; 255: not a number) as there.
#pragma once
#include "qmlp_mx.h"

namespace qmlp {

constexpr int kMx8Plane = 4096;
constexpr int kMx8Codes = 2 * kMx8Plane;
constexpr int kMx8Unit = kMx8Codes + kMxRows * 8;  // 8448
constexpr uint32_t kMx8MinExp = 7u, kMx8MaxExp = 253u;  // biased E
constexpr uint32_t kMx8HighDigit = 0x04040404u;         // from the low digit's scale bytes to the high one's
constexpr uint32_t kMx8CanonScale = 3u;                 // canonical scale byte (E + 127) less the packed one

__host__ __device__ inline size_t mx8_units_bytes(int rows, int cols) {
  return (size_t)mx_row_tiles(rows) * mx_ksb(cols) * kMx8Unit;
}

// The bits of dword d that hold bits `field` of the 16 fields of 6.
constexpr uint32_t mx8_mask(int d, uint32_t field) {
  uint32_t m = 0;
  for (int i = 0; i < 16; ++i)
    for (int b = 0; b < 6; ++b)
      if (((field >> b) & 1u) && (6 * i + b) / 32 == d) m |= 1u << ((6 * i + b) % 32);
  return m;
}
constexpr uint32_t mx8_sign(int d) { return mx8_mask(d, 32u); }
constexpr uint32_t mx8_first(int d) { return mx8_mask(d, 1u); }  // h's low bit
constexpr uint32_t mx8_upper(int d) { return mx8_mask(d, 6u); }  // h's high bits
static_assert(mx8_mask(0, 16u) == mx8_first(1) && mx8_mask(1, 16u) == mx8_first(2) && mx8_mask(2, 16u) == mx8_first(0),
              "a dword's free bits are the next one's first bits");
static_assert((mx8_upper(0) ^ mx8_upper(1) ^ mx8_upper(2)) == 0xffffffffu, "the high bits share a dword");

// Group g's half of a lane's two operands.
__device__ __forceinline__ void mx8_digits(i32x4 p, int g, i32x8& low, i32x8& high) {
#pragma unroll
  for (int d = 0; d < 3; ++d) {
    low[3 * g + d] = p[d] & (int)~mx8_first((d + 1) % 3);
    high[3 * g + d] = (p[d] & (int)mx8_sign(d)) | (p[(d + 2) % 3] & (int)mx8_first(d)) | (p[3] & (int)mx8_upper(d));
  }
}

// D += A B for 4-bit A and one digit of an 8-bit B on 32 rows x 32 columns x 64 K (mx_product's counterpart); sb:
// the digit's scale bytes, the packed ones for the low digit, kMx8HighDigit more for the high one.  A block that is
// not a number has scale 255, which makes the low digit's product one; its high digit's scale byte carries into the
// next block of the same row then, whose outputs are lost already.
template <int J>
__device__ __forceinline__ f32x16 mx8_digit_product(i32x4 a, const i32x8& digit, f32x16 c, uint32_t sa, uint32_t sb) {
  const i32x8 a8 = __builtin_shufflevector(a, i32x4{0, 0, 0, 0}, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, digit, c, 4, 2, J, (int)sa, J, (int)sb);
}

// The packed scale byte from a block's largest |x| bits (fp32).
__device__ __forceinline__ uint32_t mx8_scale_byte(uint32_t maxbits) {
  const uint32_t e = maxbits >> 23;
  return e == 255u ? kMxNan : min(max(e, kMx8MinExp), kMx8MaxExp) - kMx8CanonScale;
}
// 2^(6-E): multiplying by it is exact, but for values that round to zero.
__device__ __forceinline__ float mx8_inverse(uint32_t byte) {
  return __uint_as_float((257u - byte) << 23);  // of no use for kMxNan
}

// A value's digits: {s, q's five low bits} as a 6-bit field, and q's two high bits.  Adding 2^23 rounds the scaled
// magnitude to an integer, half to even, in the sum's low bits; 128 and more (in a block's saturating values) become
// 127.
struct Mx8Digits {
  uint32_t field, high;
};
__device__ __forceinline__ Mx8Digits mx8_digits_of(float v, float inv) {
  const uint32_t q = min(__float_as_uint(fmaf(fabsf(v), inv, 8388608.0f)), 0x4b00007fu);
  return Mx8Digits{(q & 31u) | ((__float_as_uint(v) >> 26) & ~31u), (q >> 5) & 3u};
}
// A group from the 96-bit streams of its fields and of its high bits (from bit 1 of each field on).
__device__ __forceinline__ i32x4 mx8_assemble(const uint32_t (&f)[3], const uint32_t (&h)[3]) {
  // the high digit's low bit, bit 4 of a field here, goes to bit 0 of it, 32 bits before that
  const uint32_t down[3] = {__builtin_amdgcn_alignbit(f[1], f[0], 4), __builtin_amdgcn_alignbit(f[2], f[1], 4), f[2] >> 4};
  i32x4 p;
  uint32_t upper = 0;
#pragma unroll
  for (int d = 0; d < 3; ++d) {
    const int next = (d + 1) % 3;
    p[d] = (int)((f[d] & ~mx8_first(next)) | (down[next] & mx8_first(next)));
    upper |= h[d] & mx8_upper(d);
  }
  p[3] = (int)upper;
  return p;
}

// 16 values -> one group.
__device__ __forceinline__ i32x4 mx8_group(const float (&v)[16], uint32_t byte) {
  const float inv = mx8_inverse(byte);
  uint32_t f[3] = {0, 0, 0}, h[3] = {0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const Mx8Digits q = mx8_digits_of(v[i], inv);
    const int d = 6 * i / 32, at = 6 * i % 32, dh = (6 * i + 1) / 32, ah = (6 * i + 1) % 32;
    f[d] |= q.field << at;
    h[dh] |= q.high << ah;
    if (at > 26 && d < 2) f[d + 1] |= q.field >> (32 - at);
    if (ah > 30 && dh < 2) h[dh + 1] |= q.high >> (32 - ah);
  }
  const i32x4 p = mx8_assemble(f, h);
  return byte == kMxNan ? i32x4{0, 0, 0, 0} : p;
}

// The same from four neighbouring lanes of four values each (part 0..3 of the group): all four get the group.
__device__ __forceinline__ i32x4 mx8_join(f32x4 v, int part, uint32_t byte) {
  const float inv = mx8_inverse(byte);
  uint32_t f = 0, h = 0;  // four fields, 24 bits
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const Mx8Digits q = mx8_digits_of(v[i], inv);
    f |= q.field << (6 * i);
    h |= q.high << (6 * i + 1);
  }
  auto place = [&](uint32_t v, uint32_t (&o)[3]) {
    o[0] = part == 0 ? v : part == 1 ? v << 24 : 0u;
    o[1] = part == 1 ? v >> 8 : part == 2 ? v << 16 : 0u;
    o[2] = part == 2 ? v >> 16 : part == 3 ? v << 8 : 0u;
#pragma unroll
    for (int d = 0; d < 3; ++d) {
      o[d] |= (uint32_t)__shfl_xor((int)o[d], 1);
      o[d] |= (uint32_t)__shfl_xor((int)o[d], 2);
    }
  };
  uint32_t fields[3], highs[3];
  place(f, fields);
  place(h, highs);
  const i32x4 p = mx8_assemble(fields, highs);
  return byte == kMxNan ? i32x4{0, 0, 0, 0} : p;
}

// A group's integers q.
__device__ __forceinline__ void mx8_values(i32x4 p, int (&q)[16]) {
  i32x8 low = {}, high = {};
  mx8_digits(p, 0, low, high);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int d = 6 * i / 32, at = 6 * i % 32;
    uint32_t l = (uint32_t)low[d] >> at, h = (uint32_t)high[d] >> at;
    if (at > 26) {
      l |= (uint32_t)low[d + 1] << (32 - at);
      h |= (uint32_t)high[d + 1] << (32 - at);
    }
    const int m = (int)((h & 7u) * 16u + (l & 15u));
    q[i] = (l & 32u) ? -m : m;
  }
}

// Where row `row` (of a unit) holds group g of block kb.
__device__ __forceinline__ int mx8_at(int row, int kb, int g) {
  return g * kMx8Plane + (kb >> 1) * 1024 + (row + kMxRows * (kb & 1)) * 16;
}
__device__ __forceinline__ int mx8_scale_at(int row, int kb) {
  return kMx8Codes + 4 * (row + kMxRows * (kb & 1)) + (kb >> 1);
}

__device__ __forceinline__ uint32_t abs_max16(const float (&f)[16]) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  return m;
}

// Finishes four neighbouring features n0.. of token t of row tile tt from the matrices' sums.  Packed outputs: a
// block's 32 features are eight neighbouring lanes' (item: the lane's place, item % 8 in the block).
template <int NMAT, int MODE, bool A8>
__device__ __forceinline__ void mx_finish4(const MxOut& o, int tt, int t, int n0, int item, f32x4 (&sum)[NMAT]) {
  const int m = tt * 32 + t;
  if constexpr (MODE == kMxRowsOut) {
    mx_store4(o, m, n0, sum[0]);
  } else {
    if constexpr (A8) {
      sum[0] += mx_addend(o.gate_add, o, m, n0);
      sum[NMAT - 1] += mx_addend(o.up_add, o, m, n0);
    }
    f32x4 h;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = silu_mul(sum[0][i], sum[NMAT - 1][i]);
    if constexpr (MODE == kMxGated) {
      mx_store4(o, m, n0, h);
    } else {
      uint32_t mx = 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = max(mx, __float_as_uint(h[i]) & 0x7fffffffu);
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, d));
      const int kb = (n0 % kMxK) / kMxBlock;
      const size_t u = (size_t)tt * mx_ksb(o.N) + n0 / kMxK;
      if constexpr (MODE == kMxPacked8) {
        const uint32_t s = mx8_scale_byte(mx);
        const i32x4 group = mx8_join(h, item & 3, s);
        if (m < o.M) {
          uint8_t* unit = (uint8_t*)o.out + u * kMx8Unit;
          if ((item & 3) == 0) *(i32x4*)(unit + mx8_at(t, kb, (item >> 2) & 1)) = group;
          if ((item & 7) == 0) unit[mx8_scale_at(t, kb)] = (uint8_t)s;
        }
      } else {
        const uint32_t s = mx_scale_byte(mx);
        const uint32_t c = mx_codes4(h, s);
        const uint32_t hi = (uint32_t)__shfl_xor((int)c, 1);
        if (m < o.M) {
          uint8_t* unit = (uint8_t*)o.out + u * kMxUnit;
          if ((item & 1) == 0) *(uint32_t*)(unit + (kb * 32 + t) * 16 + (n0 % kMxBlock) / 2) = c | (hi << 16);
          if ((item & 7) == 0) unit[kMxCodes + 4 * (t + 32 * (kb & 1)) + (kb >> 1)] = (uint8_t)s;
        }
      }
    }
  }
}

// 16 neighbouring values of type T (0 bf16, 1 fp16, 2 fp32; QMLP_X_*) as fp32.
template <int T>
__device__ __forceinline__ void mx8_load(const uint8_t* p, MxWords<T> (&w)[2]) {
  w[0] = mx_load8<T>(p);
  w[1] = mx_load8<T>(p + (T == 2 ? 32 : 16));
}
template <int T>
__device__ __forceinline__ void mx8_floats(const MxWords<T> (&w)[2], float (&f)[16]) {
  float a[8], b[8];
  mx_floats<T>(w[0], a);
  mx_floats<T>(w[1], b);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] = a[i];
    f[8 + i] = b[i];
  }
}

constexpr int kMx8FewTokens = 16;
int launch_mx8_few(const MxProduct& p, const MxPlan& pl, hipStream_t s);
int launch_mx8_quantize(const void* x, int type, size_t row_bytes, int rows, int cols, void* packed, hipStream_t s);
int launch_mx8_dequantize(const void* packed, int rows, int cols, void* out, bool f32, hipStream_t s);
int launch_mx8_unpack(const void* packed, int rows, int cols, void* q, void* scales, hipStream_t s);

// The norm behind the residual's addition (qmlp_add_norm.hip).  Types: QMLP_X_BF16 or QMLP_X_F32; r may be
// null (nothing is added, and h stays unwritten); h is of r's type; n (bf16) or packed may be null.
struct AddNorm {
  const uint8_t* x;
  const uint8_t* r;
  const uint16_t* w;
  uint8_t* h;
  uint16_t* n;
  uint8_t* packed;
  size_t x_bytes, r_bytes, h_bytes;  // from row to row
  float eps;
  int rows, cols, x_type, r_type;
};
int launch_add_norm(const AddNorm& a, hipStream_t s);

}  // namespace qmlp
