// qmlp_add_norm.hip -- the residual's addition and the zero-centred RMSNorm of the sum, as rows and as MXINT8
// (layout: qmlp_mx8.h).
//
//   h = T(x + r),   n = bf16(h * (1 / sqrt(mean(h^2) + eps)) * (1 + w)),   packed = MXINT8(n)
//
// T is the residual stream's type: h is rounded once, and the norm is that of the stored h, as where the
// steps are calls of their own; n is rounded to bf16 as the decoder's separate norm writes it, so that packed
// is what a quantisation of those rows makes.
//
// Bound by memory: 2048 bf16 rows of 5120 take 17.7-18.1 us (42 MB read, 32 written: 4.1 TB/s), 777 rows of an fp32
// partial on an fp32 stream 13.3 (32 and 20 MB), one row 3.9, of which nearly all is the launch.  With bf16 rows instead of
// the packed ones, captured: 15.0 us (84 MB, 5.6 TB/s), 11.1 and 3.6; with both 18.6 (95 MB, 5.1 TB/s), 13.3 and 4.5.
#include <algorithm>

#include "../../include/qwen_mlp.h"
#include "qmlp_internal.h"
#include "qmlp_mx8.h"
#include "qmlp_xcd.h"

namespace qmlp {

constexpr int kNoAdd = -1;  // RT: nothing is added

// Rounds to bf16 and back (v_cvt_pk_bf16_f32, half to even).
template <int V>
__device__ __forceinline__ void round_bf16(float (&f)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += 2) {
    const uint32_t w = mx_bf16x2(f[i], f[i + 1]);
    f[i] = __uint_as_float(w << 16);
    f[i + 1] = __uint_as_float(w & 0xffff0000u);
  }
}

// V neighbouring values of type T as fp32.
template <int T, int V>
__device__ __forceinline__ void load_values(const uint8_t* p, float (&f)[V]) {
  if constexpr (T == QMLP_X_F32) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const f32x4 v = *(const f32x4*)(p + 16 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[4 * i + j] = v[j];
    }
  } else {
    uint32_t w[V / 2];
    if constexpr (V >= 8) {
#pragma unroll
      for (int q = 0; q < V / 8; ++q) {
        const u32x4 v = *(const u32x4*)(p + 16 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[4 * q + i] = v[i];
      }
    } else {
      const u32x2 v = *(const u32x2*)p;
      w[0] = v.x;
      w[1] = v.y;
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <int T, int V>
__device__ __forceinline__ void store_values(uint8_t* p, const float (&f)[V]) {  // of type T, which holds them exactly
  if constexpr (T == QMLP_X_F32) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) *(f32x4*)(p + 16 * i) = f32x4{f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]};
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      w[i] = (__float_as_uint(f[2 * i]) >> 16) | (__float_as_uint(f[2 * i + 1]) & 0xffff0000u);
    if constexpr (V >= 8) {
#pragma unroll
      for (int q = 0; q < V / 8; ++q) *(u32x4*)(p + 16 * q) = u32x4{w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]};
    } else {
      *(u32x2*)p = u32x2{w[0], w[1]};
    }
  }
}

// The sum of a row's squares over the workgroup, in a fixed order.
__device__ __forceinline__ float row_sum(float ss, float* s_sum) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
  if ((tid & 63) == 0) s_sum[tid >> 6] = ss;
  __syncthreads();
  ss = 0.f;
  for (int i = 0; i < (int)blockDim.x / 64; ++i) ss += s_sum[i];
  return ss;
}
__device__ __forceinline__ float norm_value(float h, float rs, float w) { return h * rs * (1.0f + w); }
// Quantises one group (two neighbouring lanes a block) of row m into its unit.
__device__ __forceinline__ void store_group(uint8_t* packed, int nsb, int m, int c, bool in, const float (&f)[16]) {
  uint32_t top = abs_max16(f);
  top = max(top, (uint32_t)__shfl_xor((int)top, 1));
  const uint32_t s = mx8_scale_byte(top);
  if (!in) return;
  uint8_t* unit = packed + ((size_t)(m / kMxRows) * nsb + c / 16) * kMx8Unit;
  const int row = m % kMxRows, kb = (c / 2) % 8;
  *(i32x4*)(unit + mx8_at(row, kb, c & 1)) = mx8_group(f, s);
  if ((c & 1) == 0) unit[mx8_scale_at(row, kb)] = (uint8_t)s;
}

// One workgroup a row of up to 16384 values, 16 of them a thread in pieces of 16 bytes that neighbouring threads read
// side by side; the normalised row goes through LDS, where a thread finds 16 neighbouring values (read as such from
// memory, every lane of a load is an access of its own: 16.4 us at 777 fp32 rows of 5120).  Rows run in XCD order: 32
// rows share the lines of a packed unit, and eight XCDs writing 16 bytes of each cost 20.3 us at 2048 bf16 rows
// against 18.9.
template <int XT, int RT>
__global__ __launch_bounds__(1024) void add_norm_kernel(AddNorm a) {
  __shared__ float s_sum[16];
  extern __shared__ __align__(16) uint16_t s_row[];
  constexpr int V = XT == QMLP_X_F32 || RT == QMLP_X_F32 ? 4 : 8, kPieces = 16 / V;
  constexpr int kX = XT == QMLP_X_F32 ? 4 : 2, kR = RT == QMLP_X_F32 ? 4 : 2;  // bytes of a value
  constexpr int T = RT == kNoAdd ? 0 : RT;
  const int m = xcd_run(blockIdx.x, gridDim.x), tid = threadIdx.x, nsb = mx_ksb(a.cols), step = blockDim.x * V;
  const uint8_t* xr = a.x + (size_t)m * a.x_bytes;
  const uint8_t* rr = RT == kNoAdd ? nullptr : a.r + (size_t)m * a.r_bytes;
  uint8_t* hr = RT == kNoAdd ? nullptr : a.h + (size_t)m * a.h_bytes;
  float f[kPieces][V], r[kPieces][V], w[kPieces][V];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int k = tid * V + i * step;
#pragma unroll
    for (int j = 0; j < V; ++j) f[i][j] = r[i][j] = w[i][j] = 0.f;
    if (k < a.cols) {
      load_values<XT, V>(xr + (size_t)k * kX, f[i]);
      if constexpr (RT != kNoAdd) load_values<T, V>(rr + (size_t)k * kR, r[i]);
      load_values<QMLP_X_BF16, V>((const uint8_t*)(a.w + k), w[i]);
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int k = tid * V + i * step;
    if constexpr (RT != kNoAdd) {
#pragma unroll
      for (int j = 0; j < V; ++j) f[i][j] += r[i][j];
      if constexpr (RT == QMLP_X_BF16) round_bf16<V>(f[i]);
      if (k < a.cols) store_values<T, V>(hr + (size_t)k * kR, f[i]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) ss = fmaf(f[i][j], f[i][j], ss);
  }
  const float rs = 1.0f / sqrtf(row_sum(ss, s_sum) / (float)a.cols + a.eps);
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int k = tid * V + i * step;
    float n[V];
#pragma unroll
    for (int j = 0; j < V; ++j) n[j] = k < a.cols ? norm_value(f[i][j], rs, w[i][j]) : 0.f;
    round_bf16<V>(n);
    if (a.n && k < a.cols) store_values<QMLP_X_BF16, V>((uint8_t*)(a.n + (size_t)m * a.cols + k), n);
    if (a.packed) store_values<QMLP_X_BF16, V>((uint8_t*)(s_row + k), n);  // zeros behind the row: the padding
  }
  if (!a.packed) return;
  __syncthreads();
  float g[16];
  load_values<QMLP_X_BF16, 16>((const uint8_t*)(s_row + 16 * tid), g);
  store_group(a.packed, nsb, m, tid, tid < nsb * 16, g);
}

// Longer rows: 16 values ("a chunk") a thread at a time; the sums are read again from where they were stored (by the
// same thread): 64.7 us for 2048 bf16 rows of 17408 (3.9 TB/s without what is read again), 50.0 for rows of 16384 in
// the kernel above.
template <int XT, int RT>
__global__ __launch_bounds__(1024) void add_norm_long_kernel(AddNorm a) {
  __shared__ float s_sum[16];
  constexpr int kX = XT == QMLP_X_F32 ? 64 : 32, kR = RT == QMLP_X_F32 ? 64 : 32;  // bytes of a chunk
  constexpr int T = RT == kNoAdd ? 0 : RT;
  const int m = xcd_run(blockIdx.x, gridDim.x), tid = threadIdx.x, nch = a.cols / 16, nsb = mx_ksb(a.cols);
  const uint8_t* xr = a.x + (size_t)m * a.x_bytes;
  const uint8_t* rr = RT == kNoAdd ? nullptr : a.r + (size_t)m * a.r_bytes;
  uint8_t* hr = RT == kNoAdd ? nullptr : a.h + (size_t)m * a.h_bytes;
  float f[16], g[16], ss = 0.f;
  for (int c = tid; c < nch; c += blockDim.x) {
    load_values<XT, 16>(xr + (size_t)c * kX, f);
    if constexpr (RT != kNoAdd) {
      load_values<T, 16>(rr + (size_t)c * kR, g);
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] += g[i];
      if constexpr (RT == QMLP_X_BF16) round_bf16<16>(f);
      store_values<T, 16>(hr + (size_t)c * kR, f);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) ss = fmaf(f[i], f[i], ss);
  }
  const float rs = 1.0f / sqrtf(row_sum(ss, s_sum) / (float)a.cols + a.eps);
  for (int c0 = 0; c0 < nsb * 16; c0 += blockDim.x) {  // up to the unit's end; all lanes of a wave take part
    const int c = c0 + tid, from = min(c, nch - 1);
    load_values<QMLP_X_BF16, 16>((const uint8_t*)(a.w + (size_t)from * 16), g);
    if constexpr (RT == kNoAdd)
      load_values<XT, 16>(xr + (size_t)from * kX, f);
    else if (c < nch)  // a chunk that another thread stores is not read
      load_values<T, 16>(hr + (size_t)c * kR, f);
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = c < nch ? norm_value(f[i], rs, g[i]) : 0.f;
    round_bf16<16>(f);
    if (a.n && c < nch) store_values<QMLP_X_BF16, 16>((uint8_t*)(a.n + (size_t)m * a.cols + (size_t)c * 16), f);
    if (a.packed) store_group(a.packed, nsb, m, c, c < nsb * 16, f);
  }
}

template <int XT, int RT>
static int launch_norm(const AddNorm& a, hipStream_t s) {
  const int chunks = mx_ksb(a.cols) * 16, threads = std::min(1024, (chunks + 63) / 64 * 64);
  if (chunks <= 1024)
    hipLaunchKernelGGL((add_norm_kernel<XT, RT>), dim3(a.rows), dim3(threads), a.packed ? threads * 32 : 0, s, a);
  else
    hipLaunchKernelGGL((add_norm_long_kernel<XT, RT>), dim3(a.rows), dim3(threads), 0, s, a);
  return check_launch("add_norm_kernel");
}

template <int XT>
static int launch_stream_type(const AddNorm& a, hipStream_t s) {
  if (!a.r) return launch_norm<XT, kNoAdd>(a, s);
  if (a.r_type == QMLP_X_BF16) return launch_norm<XT, QMLP_X_BF16>(a, s);
  return launch_norm<XT, QMLP_X_F32>(a, s);
}

int launch_add_norm(const AddNorm& a, hipStream_t s) {
  return a.x_type == QMLP_X_BF16 ? launch_stream_type<QMLP_X_BF16>(a, s) : launch_stream_type<QMLP_X_F32>(a, s);
}

}  // namespace qmlp
