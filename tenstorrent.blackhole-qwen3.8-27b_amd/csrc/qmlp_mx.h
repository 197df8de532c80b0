// qmlp_mx.h -- the MXFP4 format (microscaled 4-bit floating point): layout and device helpers.
//
// A matrix X[rows, K] in the format: 32 consecutive K values share one scale 2^(s - 127) (a byte s;
// 255 marks a block that is not a number), each value is one of 0, .5, 1, 1.5, 2, 3, 4, 6 with a sign
// (e2m1: code = sign * 8 + index).  Weights and activations use the same packed layout:
//   * units of 32 rows x 256 K, unit index u = (row / 32) * ceil(K / 256) + K / 256, 4352 B each;
//   * codes: the 16 bytes of block kb = (k % 256) / 32 of row r % 32 at (kb * 32 + r % 32) * 16, two
//     codes to a byte, the even K in the low half;
//   * scales: 64 dwords at 4096; dword (r % 32) + 32 * (kb % 2) holds, in byte kb / 2, block kb's scale.
// So lane l of a wave reads the operand of the 32x32x64 scaled product of K-step j (64 K values) as 16
// bytes at 1024 j + 16 l -- row l % 32, block 2 j + l / 32 -- and the scales of all four steps of a
// unit as dword l, whose byte j the product selects by itself.  Rows behind the last one of an
// activation matrix are not written (they are token columns that no output uses); K behind the last
// block up to the unit's end holds zeros with a finite scale, on both sides.
#pragma once
#include "qmlp_common.h"

namespace qmlp {

constexpr int kMxRows = 32;
constexpr int kMxK = 256;
constexpr int kMxBlock = 32;
constexpr int kMxCodes = kMxRows * kMxK / 2;     // 4096
constexpr int kMxUnit = kMxCodes + kMxRows * 8;  // 4352
constexpr int kMxPackedX = 3;  // QMLP_X_MXFP4
constexpr uint32_t kMxNan = 255u;
constexpr uint32_t kMxMinScale = 1u;  // 2^-126: the smallest scale that is a normal fp32 number

__host__ __device__ inline int mx_ksb(int cols) { return (cols + kMxK - 1) / kMxK; }
__host__ __device__ inline int mx_row_tiles(int rows) { return (rows + kMxRows - 1) / kMxRows; }
__host__ __device__ inline size_t mx_units_bytes(int rows, int cols) {
  return (size_t)mx_row_tiles(rows) * mx_ksb(cols) * kMxUnit;
}

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// The scale byte of a block from the largest |x| bits (fp32) in it: the binade of the maximum less 2,
// so that it lands in [4, 8) (values from 5 up to 8 become 4 or 6); at least kMxMinScale.  An infinity
// or a NaN in the block makes the whole block one.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t maxbits) {
  const uint32_t e = maxbits >> 23;
  return e == 255u ? kMxNan : max(e, kMxMinScale + 2u) - 2u;
}

// 8 fp32 values -> 8 codes, rounded half to even and saturated at 6 by the hardware conversion
// (v_cvt_scalef32_pk_fp4_f32, compared with the definition for every bf16 value at scales from 2^-127
// to 2^125).
__device__ __forceinline__ uint32_t mx_codes8(const float (&v)[8], uint32_t byte) {
  const float s = __uint_as_float(byte << 23);
  uint32_t o = 0u;
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[0], v[1], s, 0);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[2], v[3], s, 1);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[4], v[5], s, 2);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[6], v[7], s, 3);
  return byte == kMxNan ? 0u : o;
}

// 4 fp32 values -> 4 codes in the low 16 bits, as mx_codes8.
__device__ __forceinline__ uint32_t mx_codes4(f32x4 v, uint32_t byte) {
  const float s = __uint_as_float(byte << 23);
  uint32_t o = 0u;
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v.x, v.y, s, 0);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v.z, v.w, s, 1);
  return byte == kMxNan ? 0u : o;
}

// ---------------------------------------------------------------- 8 values of a row
//
// Four neighbouring lanes own a block, 8 values each.
__device__ __forceinline__ uint32_t max4(uint32_t v) {  // over the block's four lanes
  v = max(v, (uint32_t)__shfl_xor((int)v, 1));
  return max(v, (uint32_t)__shfl_xor((int)v, 2));
}

// T: 0 bf16, 1 fp16, 2 fp32 (QMLP_X_*)
template <int T>
struct MxWords {
  u32x4 w[T == 2 ? 2 : 1];
};
template <int T>
__device__ __forceinline__ MxWords<T> mx_load8(const uint8_t* p) {
  MxWords<T> v;
  v.w[0] = *(const u32x4*)p;
  if constexpr (T == 2) v.w[1] = *(const u32x4*)(p + 16);
  return v;
}
template <int T>
__device__ __forceinline__ void mx_floats(const MxWords<T>& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T == 0) {
      f[2 * i] = __uint_as_float(v.w[0][i] << 16);
      f[2 * i + 1] = __uint_as_float(v.w[0][i] & 0xffff0000u);
    } else if constexpr (T == 1) {
      const f16x2 h = as_f16x2(v.w[0][i]);
      f[2 * i] = (float)h.x;
      f[2 * i + 1] = (float)h.y;
    } else {
      f[i] = __uint_as_float(v.w[0][i]);
      f[4 + i] = __uint_as_float(v.w[1][i]);
    }
  }
}
__device__ __forceinline__ uint32_t abs_max8(const float (&f)[8]) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  return m;
}

// D += A B on 32 rows x 32 columns x 64 K; J: the step inside a unit, whose scales are byte J of each
// lane's scale dword.
template <int J>
__device__ __forceinline__ f32x16 mx_product(i32x4 a, i32x4 b, f32x16 c, uint32_t sa, uint32_t sb) {
  const i32x8 a8 = __builtin_shufflevector(a, i32x4{0, 0, 0, 0}, 0, 1, 2, 3, 4, 5, 6, 7);
  const i32x8 b8 = __builtin_shufflevector(b, i32x4{0, 0, 0, 0}, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, J, (int)sa, J, (int)sb);
}

// ---------------------------------------------------------------- epilogues shared by the products

// What a product kernel leaves behind.
constexpr int kMxRowsOut = 0;  // out[m, n] = sum (+ residual), bf16 or fp32
constexpr int kMxGated = 1;    // out[m, n] = silu(gate) * up, bf16 or fp32
constexpr int kMxPacked = 2;   // the same, quantised into a packed activation matrix
constexpr int kMxPacked8 = 3;  // the same, as MXINT8 (qmlp_mx8.h)

struct MxOut {
  void* out;
  const void* residual;  // kMxRowsOut only, may be null
  int M, N;
  int out_f32, res_f32;
  const float* gate_add;  // gated modes of 8-bit activations: fp32 [M, N] added to the matrices' sums in
  const float* up_add;    // front of the SiLU, may be null
};

// One product: packed activations x [M, K] times one packed weight matrix [N, K], or two of them.
struct MxProduct {
  const uint8_t* x;  // packed, or with x_type < QMLP_X_MXFP4 rows that the product kernel quantises
  const uint8_t* w0;
  const uint8_t* w1;  // up (gated modes)
  int K, mode;
  MxOut o;
  int slot;  // launch_timed's slot, -1: not timed
  int x_type;        // QMLP_X_*
  size_t row_bytes;  // of unpacked rows
  void* parts;       // kMxPartBytes for the partial tiles of split K ranges (many tokens)
  bool a8;           // activations in 8 bits (MXINT8) instead of 4
};
constexpr size_t kMxPartBytes = 64u << 20;
constexpr int kMxInside = 4;  // at most this many token rows are quantised inside the streamed product
bool mx_quantizes_inside(int M, int K, bool a8);
constexpr int kMxFewTokens = 32;  // up to here no product is tiled: streamed, or (8-bit activations) the few-token kernel's

// How a product runs (mx_plan, qmlp_mx_plan.hip).  Streamed: a workgroup of 32 features x 32 tokens, four
// waves with one unit of K under way (kMxStream) or two (kMxStreamDeep, one matrix only), or eight with
// two (kMxStreamLong); or of 32 features x 64 tokens (kMxStreamWide).  Tiled (kMxTiles): 256 features (128
// of gate and up each) x 64 height tokens a workgroup, the K range in ks pieces but for the first `whole` tiles.
// Up to 16 tokens of 8-bit activations have a kernel of their own (kMxFew, height: its waves where it quantises rows).
enum MxKind { kMxStream, kMxStreamDeep, kMxStreamLong, kMxStreamWide, kMxTiles, kMxFew };
struct MxPlan {
  MxKind kind;
  int height, ks;
  int workgroups;
  size_t part_bytes;  // of all pieces
  int whole;
};
MxPlan mx_plan(int M, int N, int K, int nmat, int num_cus, bool a8);
int launch_mx_stream(const MxProduct& p, const MxPlan& pl, hipStream_t s);
int launch_mx_tiled(const MxProduct& p, const MxPlan& pl, hipStream_t s);
int launch_mx_quantize(const void* x, int type, size_t row_bytes, int rows, int cols, void* packed, hipStream_t s);
int launch_mx_norm_quantize(const void* x, size_t row_bytes, const void* w, float eps, int rows, int cols,
                            void* packed, hipStream_t s);
int launch_mx_quantize_pack(const void* w, int rows, int cols, void* packed, hipStream_t s);
int launch_mx_pack(const void* codes, const void* scales, int rows, int cols, void* packed, hipStream_t s);
int launch_mx_unpack(const void* packed, int rows, int cols, void* codes, void* scales, hipStream_t s);
int launch_mx_dequantize(const void* packed, int rows, int cols, void* out, bool f32, hipStream_t s);

// Two fp32 values -> bf16, rounded half to even (v_cvt_pk_bf16_f32, one instruction where the word
// arithmetic of f32_to_bf16 takes a dozen).
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t mx_bf16x2(float a, float b) {
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}

// Four neighbouring features of an fp32 [M, N] matrix that is added to a product's sums.
__device__ __forceinline__ f32x4 mx_addend(const float* p, const MxOut& o, int m, int n) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (!p || m >= o.M || n >= o.N) return v;
  p += (size_t)m * o.N + n;
  if ((o.N & 3) == 0) return *(const f32x4*)p;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < o.N) v[i] = p[i];
  return v;
}

// Four neighbouring features n..n+3 of token m.  N may be any number: rows whose length is not a
// multiple of 4 start misaligned for vector stores.
__device__ __forceinline__ void mx_store4(const MxOut& o, int m, int n, f32x4 v) {
  if (m >= o.M || n >= o.N) return;
  const size_t at = (size_t)m * o.N + n;
  if ((o.N & 3) == 0) {
    if (o.residual) {
      if (o.res_f32) {
        v += *(const f32x4*)((const float*)o.residual + at);
      } else {
        const u32x2 r = *(const u32x2*)((const uint16_t*)o.residual + at);
        v += f32x4{__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16),
                   __uint_as_float(r.y & 0xffff0000u)};
      }
    }
    if (o.out_f32) {
      *(f32x4*)((float*)o.out + at) = v;
    } else {
      *(u32x2*)((uint16_t*)o.out + at) =
          u32x2{mx_bf16x2(v.x, v.y), mx_bf16x2(v.z, v.w)};
    }
    return;
  }
  for (int i = 0; i < 4 && n + i < o.N; ++i) {
    float f = v[i];
    if (o.residual)
      f += o.res_f32 ? ((const float*)o.residual)[at + i] : bf16_to_f32(((const uint16_t*)o.residual)[at + i]);
    if (o.out_f32)
      ((float*)o.out)[at + i] = f;
    else
      ((uint16_t*)o.out)[at + i] = f32_to_bf16(f);
  }
}

}  // namespace qmlp
