// qmlp_mx_pack.hip -- MXFP4 quantisation of activations and weights, packing, unpacking and
// dequantisation (layout: qmlp_mx.h).
#include "qmlp_internal.h"
#include "qmlp_mx.h"

namespace qmlp {

// ---------------------------------------------------------------- thread mapping
//
// Four neighbouring lanes own a 32-value block, 8 values each.  A wave covers 8 rows x 2 blocks, so a
// read touches 128 contiguous bytes of a row (16-bit values) and a write 128 contiguous bytes of the
// packed codes; a workgroup of four waves covers 8 rows x 256 K, R times (R * 8 rows).
constexpr int kQThreads = 256;

struct MxItem {
  int p;   // which 8 values of the block
  int r;   // row inside the group of 8
  int kb;  // block inside the unit
};
__device__ __forceinline__ MxItem mx_item(int tid) {
  return MxItem{tid & 3, (tid >> 2) & 7, (tid >> 6) * 2 + ((tid >> 5) & 1)};
}

// ---------------------------------------------------------------- quantisation
//
// Bound by memory for many rows (2 or 4 bytes read and 17/32 written per value: 2048 x 17408 bf16 in
// 14.0-16.4 us, 5.5-6.4 TB/s), by latency for few (one row of 5120: 2.4-2.6 us).
// R groups of 8 rows keep R 16-byte loads of a thread in flight.  The scale bytes of a workgroup
// gather in LDS, so that they leave as whole dwords.  Rows [rows, fill_rows) are written as zeros
// (weights, whose packed bytes depend on the weights alone); bad (weights): count of blocks that hold
// a value that is not finite.
template <int T, int R>
__global__ __launch_bounds__(kQThreads) void mx_quantize_kernel(const uint8_t* __restrict__ x, size_t row_bytes,
                                                               int rows, int cols, int fill_rows,
                                                               uint8_t* __restrict__ packed, uint32_t* bad) {
  __shared__ uint8_t s_scale[R * 8 * 8];  // [R][row][kb % 2][kb / 2]
  const MxItem it = mx_item(threadIdx.x);
  const int sb = blockIdx.x, nsb = gridDim.x;
  const int row0 = blockIdx.y * (8 * R);
  const int k = sb * kMxK + it.kb * kMxBlock + it.p * 8;
  MxWords<T> v[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = row0 + i * 8 + it.r;
    if (row < rows && k < cols)
      v[i] = mx_load8<T>(x + (size_t)row * row_bytes + (size_t)k * (T == 2 ? 4 : 2));
    else
      v[i] = MxWords<T>{};
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float f[8];
    mx_floats<T>(v[i], f);
    const uint32_t s = mx_scale_byte(max4(abs_max8(f)));
    const uint32_t code = mx_codes8(f, s);
    const int row = row0 + i * 8 + it.r;
    if (row < fill_rows) {
      uint8_t* unit = packed + ((size_t)(row / kMxRows) * nsb + sb) * kMxUnit;
      *(uint32_t*)(unit + (it.kb * kMxRows + row % kMxRows) * 16 + it.p * 4) = code;
    }
    if (it.p == 0) {
      s_scale[(i * 8 + it.r) * 8 + (it.kb & 1) * 4 + (it.kb >> 1)] = (uint8_t)s;
      if (bad && s == kMxNan) atomicAdd(bad, 1u);
    }
  }
  __syncthreads();
  if (threadIdx.x < R * 16) {
    const int row = row0 + threadIdx.x / 2, half = threadIdx.x & 1;
    if (row < fill_rows) {
      uint8_t* unit = packed + ((size_t)(row / kMxRows) * nsb + sb) * kMxUnit;
      *(uint32_t*)(unit + kMxCodes + 4 * (row % kMxRows + kMxRows * half)) =
          *(const uint32_t*)(s_scale + threadIdx.x * 4);
    }
  }
}

template <int T>
static int launch_quant(const void* x, size_t row_bytes, int rows, int cols, int fill_rows, void* packed,
                        uint32_t* bad, hipStream_t s) {
  const int nsb = mx_ksb(cols);
  // four row groups a workgroup once that still leaves a few workgroups for every CU
  const bool tall = (size_t)nsb * ((fill_rows + 31) / 32) >= 1024;
  const int step = tall ? 32 : 8;
  const dim3 grid(nsb, (fill_rows + step - 1) / step);
  auto kern = tall ? mx_quantize_kernel<T, 4> : mx_quantize_kernel<T, 1>;
  hipLaunchKernelGGL(kern, grid, dim3(kQThreads), 0, s, (const uint8_t*)x, row_bytes, rows, cols, fill_rows,
                     (uint8_t*)packed, bad);
  return check_launch("mx_quantize_kernel");
}

int launch_mx_quantize(const void* x, int type, size_t row_bytes, int rows, int cols, void* packed, hipStream_t s) {
  if (type == 0) return launch_quant<0>(x, row_bytes, rows, cols, rows, packed, nullptr, s);
  if (type == 1) return launch_quant<1>(x, row_bytes, rows, cols, rows, packed, nullptr, s);
  return launch_quant<2>(x, row_bytes, rows, cols, rows, packed, nullptr, s);
}

// ---------------------------------------------------------------- RMSNorm in front
//
// The decoder's zero-centred norm, n = bf16(x * (1 / sqrt(mean(x^2) + eps)) * (1 + w)), then n's blocks.
// One workgroup per row, the sums in rows_kernel's order, so that the result is that of the norm pass
// followed by the quantisation, bit for bit.  Bound by latency (a row's load, a reduction, its store)
// for few rows: 3.4-4.6 us at 16 of 5120 values.  For many its stores bound it, 4 bytes in runs of 16 and
// single scale bytes: 7.6 us at 777 rows, 11.0 at 2048 (2.4 TB/s), where the quantisation alone, whose
// workgroups write whole dwords of eight rows, takes 8.7.  REGS: rows of up to 8192 values stay in registers.
constexpr int kNormCh = 4;
template <bool REGS>
__global__ __launch_bounds__(kQThreads) void mx_norm_quantize_kernel(const uint8_t* __restrict__ x, size_t row_bytes,
                                                                    const uint16_t* __restrict__ w, float eps,
                                                                    int cols, uint8_t* __restrict__ packed) {
  __shared__ float s_sum[4];
  const int m = blockIdx.x, nch = cols / 8, tid = threadIdx.x, nsb = mx_ksb(cols);
  const u32x4* xr = (const u32x4*)(x + (size_t)m * row_bytes);
  const u32x4* wr = (const u32x4*)w;
  u32x4 v[REGS ? kNormCh : 1], g[REGS ? kNormCh : 1];
  if constexpr (REGS) {
#pragma unroll
    for (int i = 0; i < kNormCh; ++i) {
      const int c = min(tid + i * kQThreads, nch - 1);
      v[i] = xr[c];
      g[i] = wr[c];
    }
  }
  float ss = 0.f;
  auto add = [&](const u32x4& t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = __uint_as_float(t[i] << 16), b = __uint_as_float(t[i] & 0xffff0000u);
      ss = fmaf(a, a, ss);
      ss = fmaf(b, b, ss);
    }
  };
  if constexpr (REGS) {
#pragma unroll
    for (int i = 0; i < kNormCh; ++i)
      if (tid + i * kQThreads < nch) add(v[i]);
  } else {
    for (int c = tid; c < nch; c += kQThreads) add(xr[c]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
  if ((tid & 63) == 0) s_sum[tid >> 6] = ss;
  __syncthreads();
  ss = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
  const float rs = 1.0f / sqrtf(ss / (float)cols + eps);
  uint8_t* rowp = packed + (size_t)(m / kMxRows) * nsb * kMxUnit;
  // chunk c (8 values) of the row: every lane of a wave takes part, a chunk at or behind nch as zeros
  // (up to the unit's end they are the padding)
  auto emit = [&](int c, const u32x4& t, const u32x4& u) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = __uint_as_float(t[i] << 16) * rs * (1.0f + __uint_as_float(u[i] << 16));
      const float b = __uint_as_float(t[i] & 0xffff0000u) * rs * (1.0f + __uint_as_float(u[i] & 0xffff0000u));
      f[2 * i] = c < nch ? bf16_to_f32(f32_to_bf16(a)) : 0.f;
      f[2 * i + 1] = c < nch ? bf16_to_f32(f32_to_bf16(b)) : 0.f;
    }
    const uint32_t s = mx_scale_byte(max4(abs_max8(f)));
    const uint32_t code = mx_codes8(f, s);
    if (c < nsb * 32) {
      uint8_t* unit = rowp + (size_t)(c / 32) * kMxUnit;
      const int kb = (c / 4) % 8, row = m % kMxRows;
      *(uint32_t*)(unit + (kb * kMxRows + row) * 16 + (c & 3) * 4) = code;
      if ((c & 3) == 0) unit[kMxCodes + 4 * (row + kMxRows * (kb & 1)) + (kb >> 1)] = (uint8_t)s;
    }
  };
  if constexpr (REGS) {
#pragma unroll
    for (int i = 0; i < kNormCh; ++i)
      if (i * kQThreads < nsb * 32) emit(tid + i * kQThreads, v[i], g[i]);
  } else {
    for (int c0 = 0; c0 < nsb * 32; c0 += kQThreads) {
      const int c = min(c0 + tid, nch - 1);
      emit(c0 + tid, xr[c], wr[c]);
    }
  }
}

int launch_mx_norm_quantize(const void* x, size_t row_bytes, const void* w, float eps, int rows, int cols,
                            void* packed, hipStream_t s) {
  auto kern = cols <= 8 * kQThreads * kNormCh ? mx_norm_quantize_kernel<true> : mx_norm_quantize_kernel<false>;
  hipLaunchKernelGGL(kern, dim3(rows), dim3(kQThreads), 0, s, (const uint8_t*)x, row_bytes, (const uint16_t*)w, eps,
                     cols, (uint8_t*)packed);
  return check_launch("mx_norm_quantize_kernel");
}

// ---------------------------------------------------------------- weights: trailer, pack, unpack

__global__ void mx_trailer_kernel(uint32_t* t) {
  if (threadIdx.x < kTrailer / 4) t[threadIdx.x] = threadIdx.x == 3 ? kTrailerMagic : 0u;
}

static int launch_mx_trailer(int rows, int cols, void* packed, hipStream_t s) {
  hipLaunchKernelGGL(mx_trailer_kernel, dim3(1), dim3(64), 0, s, (uint32_t*)((uint8_t*)packed + mx_units_bytes(rows, cols)));
  return check_launch("mx_trailer_kernel");
}

int launch_mx_quantize_pack(const void* w, int rows, int cols, void* packed, hipStream_t s) {
  if (int rc = launch_mx_trailer(rows, cols, packed, s)) return rc;
  PackTrailer* t = (PackTrailer*)((uint8_t*)packed + mx_units_bytes(rows, cols));
  return launch_quant<0>(w, (size_t)cols * 2, rows, cols, mx_row_tiles(rows) * kMxRows, packed, &t->bad_groups, s);
}

// Canonical (codes [rows, cols / 2], scales [rows, cols / 32]) <-> packed, one dword of codes a thread.
template <bool PACK>
__global__ __launch_bounds__(kQThreads) void mx_repack_kernel(uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                             int rows, int cols, uint8_t* __restrict__ packed,
                                                             uint32_t* bad) {
  const MxItem it = mx_item(threadIdx.x);
  const int sb = blockIdx.y, nsb = gridDim.y, row = blockIdx.x * 8 + it.r;
  const int kblk = sb * 8 + it.kb;
  const bool in = row < rows && kblk * kMxBlock < cols;
  uint8_t* unit = packed + ((size_t)(row / kMxRows) * nsb + sb) * kMxUnit;
  uint32_t* pc = (uint32_t*)(unit + (it.kb * kMxRows + row % kMxRows) * 16 + it.p * 4);
  uint8_t* ps = unit + kMxCodes + 4 * (row % kMxRows + kMxRows * (it.kb & 1)) + (it.kb >> 1);
  uint32_t* cc = (uint32_t*)(codes + (size_t)row * (cols / 2) + (size_t)kblk * 16 + it.p * 4);
  uint8_t* cs = scales + (size_t)row * (cols / kMxBlock) + kblk;
  if constexpr (PACK) {
    *pc = in ? *cc : 0u;
    if (it.p == 0) {
      const uint8_t b = in ? *cs : (uint8_t)kMxMinScale;
      *ps = b;
      if (b == kMxNan) atomicAdd(bad, 1u);
    }
  } else if (in) {
    *cc = *pc;
    if (it.p == 0) *cs = *ps;
  }
}

template <bool PACK>
static int launch_repack(const void* codes, const void* scales, int rows, int cols, const void* packed, uint32_t* bad,
                         hipStream_t s) {
  const dim3 grid(mx_row_tiles(rows) * 4, mx_ksb(cols));
  hipLaunchKernelGGL(mx_repack_kernel<PACK>, grid, dim3(kQThreads), 0, s, (uint8_t*)codes, (uint8_t*)scales, rows,
                     cols, (uint8_t*)packed, bad);
  return check_launch("mx_repack_kernel");
}

int launch_mx_pack(const void* codes, const void* scales, int rows, int cols, void* packed, hipStream_t s) {
  if (int rc = launch_mx_trailer(rows, cols, packed, s)) return rc;
  PackTrailer* t = (PackTrailer*)((uint8_t*)packed + mx_units_bytes(rows, cols));
  return launch_repack<true>(codes, scales, rows, cols, packed, &t->bad_groups, s);
}

int launch_mx_unpack(const void* packed, int rows, int cols, void* codes, void* scales, hipStream_t s) {
  return launch_repack<false>(codes, scales, rows, cols, packed, nullptr, s);
}

// ---------------------------------------------------------------- dequantisation
//
// Packed -> bf16 or fp32 values, exactly: a code has two significant bits, and 2^-128, the smallest
// magnitude (scale byte 0, which packed checkpoints may hold), is a bf16 number too.  Magnitudes from
// 2^128 on, which scale bytes 253 and 254 of a checkpoint can name, become infinities.  Bound by the
// write (2048 x 17408 to bf16 in 16.0-18.4 us, 4.9-5.7 TB/s); the thread mapping is the quantiser's.
template <bool F32, int R>
__global__ __launch_bounds__(kQThreads) void mx_dequantize_kernel(const uint8_t* __restrict__ packed, int rows,
                                                                 int cols, uint8_t* __restrict__ out) {
  const MxItem it = mx_item(threadIdx.x);
  const int sb = blockIdx.x, nsb = gridDim.x, row0 = blockIdx.y * (8 * R);
  const int k = sb * kMxK + it.kb * kMxBlock + it.p * 8;
  uint32_t code[R], byte[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = min(row0 + i * 8 + it.r, rows - 1);
    const uint8_t* unit = packed + ((size_t)(row / kMxRows) * nsb + sb) * kMxUnit;
    code[i] = *(const uint32_t*)(unit + (it.kb * kMxRows + row % kMxRows) * 16 + it.p * 4);
    byte[i] = unit[kMxCodes + 4 * (row % kMxRows + kMxRows * (it.kb & 1)) + (it.kb >> 1)];
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = row0 + i * 8 + it.r;
    if (row >= rows || k >= cols) continue;
    const float s = __uint_as_float(byte[i] == kMxNan ? 0x7fc00000u : byte[i] == 0u ? 0x00400000u : byte[i] << 23);
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t c = (code[i] >> (4 * j)) & 15u, e = (c >> 1) & 3u, h = c & 1u;
      const float a = e ? __uint_as_float(((126u + e) << 23) | (h << 22)) : 0.5f * (float)h;
      f[j] = __uint_as_float(__float_as_uint(a) | ((c & 8u) << 28)) * s;
    }
    uint8_t* o = out + ((size_t)row * cols + k) * (F32 ? 4 : 2);
    if constexpr (F32) {
      *(f32x4*)o = f32x4{f[0], f[1], f[2], f[3]};
      *(f32x4*)(o + 16) = f32x4{f[4], f[5], f[6], f[7]};
    } else {
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = (__float_as_uint(f[2 * j]) >> 16) | (__float_as_uint(f[2 * j + 1]) & 0xffff0000u);
      *(u32x4*)o = v;
    }
  }
}

int launch_mx_dequantize(const void* packed, int rows, int cols, void* out, bool f32, hipStream_t s) {
  const int nsb = mx_ksb(cols);
  const bool tall = (size_t)nsb * ((rows + 31) / 32) >= 1024;
  const int step = tall ? 32 : 8;
  const dim3 grid(nsb, (rows + step - 1) / step);
  auto kern = f32 ? (tall ? mx_dequantize_kernel<true, 4> : mx_dequantize_kernel<true, 1>)
                  : (tall ? mx_dequantize_kernel<false, 4> : mx_dequantize_kernel<false, 1>);
  hipLaunchKernelGGL(kern, grid, dim3(kQThreads), 0, s, (const uint8_t*)packed, rows, cols, (uint8_t*)out);
  return check_launch("mx_dequantize_kernel");
}

}  // namespace qmlp
