// qmlp_mx8_pack.hip -- MXINT8 quantisation of activations, and back (layout: qmlp_mx8.h).
#include "qmlp_internal.h"
#include "qmlp_mx8.h"

namespace qmlp {

// Two neighbouring lanes own a 32-value block, 16 values each.  A wave covers 8 rows x 4 blocks, so a read
// touches 256 contiguous bytes of a row (16-bit values) and a write 128 contiguous bytes of a plane; a
// workgroup of four waves covers 16 rows x 256 K, R times (R * 16 rows).  Bound by memory: 20-22 us for 2048 x 17408
// bf16 values (71 MB in, 37 out, 5.1 TB/s, which is the rate of a large copy), 7 for 777 x 5120 fp16, 3-4 for 16.
constexpr int kQ8Threads = 256;
constexpr int kQ8Rows = 16;

struct Mx8Item {
  int g;   // group of the block
  int kb;  // block inside the unit
  int r;   // row of the 16
};
__device__ __forceinline__ Mx8Item mx8_item(int tid) {
  return Mx8Item{tid & 1, ((tid >> 1) & 3) + ((tid >> 4) & 4), ((tid >> 3) & 7) + ((tid >> 4) & 8)};
}

template <int T, int R>
__global__ __launch_bounds__(kQ8Threads) void mx8_quantize_kernel(const uint8_t* __restrict__ x, size_t row_bytes,
                                                                 int rows, int cols, uint8_t* __restrict__ packed) {
  __shared__ uint8_t s_scale[R * kQ8Rows * 8];  // [R][row][kb % 2][kb / 2]
  const Mx8Item it = mx8_item(threadIdx.x);
  const int sb = blockIdx.x, nsb = gridDim.x, row0 = blockIdx.y * (kQ8Rows * R);
  const int k = sb * kMxK + it.kb * kMxBlock + it.g * 16;
  MxWords<T> v[R][2];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = row0 + i * kQ8Rows + it.r;
    if (row < rows && k < cols)
      mx8_load<T>(x + (size_t)row * row_bytes + (size_t)k * (T == 2 ? 4 : 2), v[i]);
    else
      v[i][0] = v[i][1] = MxWords<T>{};
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    float f[16];
    mx8_floats<T>(v[i], f);
    uint32_t top = abs_max16(f);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    const uint32_t s = mx8_scale_byte(top);
    const int row = row0 + i * kQ8Rows + it.r;
    if (row < rows)
      *(i32x4*)(packed + ((size_t)(row / kMxRows) * nsb + sb) * kMx8Unit + mx8_at(row % kMxRows, it.kb, it.g)) =
          mx8_group(f, s);
    if (it.g == 0) s_scale[(i * kQ8Rows + it.r) * 8 + (it.kb & 1) * 4 + (it.kb >> 1)] = (uint8_t)s;
  }
  __syncthreads();
  if (threadIdx.x < R * kQ8Rows * 2) {
    const int row = row0 + threadIdx.x / 2, half = threadIdx.x & 1;
    if (row < rows)
      *(uint32_t*)(packed + ((size_t)(row / kMxRows) * nsb + sb) * kMx8Unit + kMx8Codes +
                   4 * (row % kMxRows + kMxRows * half)) = *(const uint32_t*)(s_scale + threadIdx.x * 4);
  }
}

template <int T>
static int launch_quant8(const void* x, size_t row_bytes, int rows, int cols, void* packed, hipStream_t s) {
  const int nsb = mx_ksb(cols);
  const bool tall = (size_t)nsb * mx_row_tiles(rows) >= 1024;
  const int step = tall ? 2 * kQ8Rows : kQ8Rows;
  auto kern = tall ? mx8_quantize_kernel<T, 2> : mx8_quantize_kernel<T, 1>;
  hipLaunchKernelGGL(kern, dim3(nsb, (rows + step - 1) / step), dim3(kQ8Threads), 0, s, (const uint8_t*)x, row_bytes,
                     rows, cols, (uint8_t*)packed);
  return check_launch("mx8_quantize_kernel");
}

int launch_mx8_quantize(const void* x, int type, size_t row_bytes, int rows, int cols, void* packed, hipStream_t s) {
  if (type == 0) return launch_quant8<0>(x, row_bytes, rows, cols, packed, s);
  if (type == 1) return launch_quant8<1>(x, row_bytes, rows, cols, packed, s);
  return launch_quant8<2>(x, row_bytes, rows, cols, packed, s);
}

// Packed -> values (MODE 0 bf16, 1 fp32) exactly: q has seven significant bits and its step is at least 2^-126;
// or (MODE 2) -> canonical integers [rows, cols] and scale bytes E + 127 [rows, cols / 32].  2048 x 5120 to bf16: 8 us
// (32 MB, bound by its writes), one row 3.
template <int MODE>
__global__ __launch_bounds__(kQ8Threads) void mx8_read_kernel(const uint8_t* __restrict__ packed, int rows, int cols,
                                                             uint8_t* __restrict__ out, uint8_t* __restrict__ scales) {
  const Mx8Item it = mx8_item(threadIdx.x);
  const int sb = blockIdx.x, nsb = gridDim.x, row = blockIdx.y * kQ8Rows + it.r;
  const int k = sb * kMxK + it.kb * kMxBlock + it.g * 16;
  if (row >= rows || k >= cols) return;
  const uint8_t* unit = packed + ((size_t)(row / kMxRows) * nsb + sb) * kMx8Unit;
  const i32x4 p = *(const i32x4*)(unit + mx8_at(row % kMxRows, it.kb, it.g));
  const uint32_t byte = unit[mx8_scale_at(row % kMxRows, it.kb)];
  int q[16];
  mx8_values(p, q);
  if constexpr (MODE == 2) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i] = (q[4 * i] & 255u) | (q[4 * i + 1] & 255u) << 8 | (q[4 * i + 2] & 255u) << 16 | (uint32_t)q[4 * i + 3] << 24;
    *(u32x4*)(out + (size_t)row * cols + k) = o;
    if (it.g == 0)
      scales[(size_t)row * (cols / kMxBlock) + k / kMxBlock] =
          (uint8_t)(byte == kMxNan ? kMxNan : byte + kMx8CanonScale);
  } else {
    const float step = __uint_as_float(byte == kMxNan ? 0x7fc00000u : (byte - 3u) << 23);  // 2^(E-6)
    uint8_t* o = out + ((size_t)row * cols + k) * (MODE ? 4 : 2);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = (float)q[8 * h + i] * step;
      if constexpr (MODE == 1) {
        *(f32x4*)(o + 32 * h) = f32x4{f[0], f[1], f[2], f[3]};
        *(f32x4*)(o + 32 * h + 16) = f32x4{f[4], f[5], f[6], f[7]};
      } else {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[i] = (__float_as_uint(f[2 * i]) >> 16) | (__float_as_uint(f[2 * i + 1]) & 0xffff0000u);
        *(u32x4*)(o + 16 * h) = v;
      }
    }
  }
}

template <int MODE>
static int launch_read8(const void* packed, int rows, int cols, void* out, void* scales, hipStream_t s) {
  hipLaunchKernelGGL(mx8_read_kernel<MODE>, dim3(mx_ksb(cols), (rows + kQ8Rows - 1) / kQ8Rows), dim3(kQ8Threads), 0, s,
                     (const uint8_t*)packed, rows, cols, (uint8_t*)out, (uint8_t*)scales);
  return check_launch("mx8_read_kernel");
}

int launch_mx8_dequantize(const void* packed, int rows, int cols, void* out, bool f32, hipStream_t s) {
  return f32 ? launch_read8<1>(packed, rows, cols, out, nullptr, s) : launch_read8<0>(packed, rows, cols, out, nullptr, s);
}

int launch_mx8_unpack(const void* packed, int rows, int cols, void* q, void* scales, hipStream_t s) {
  return launch_read8<2>(packed, rows, cols, q, scales, s);
}

}  // namespace qmlp
