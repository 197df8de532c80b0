// qmlp_add_norm.hip -- the residual's addition and the zero-centred RMSNorm of the sum, as rows and as MXINT8
// (layout: qmlp_mx8.h).
//
//   h = T(x + r),   n = bf16(h * (1 / sqrt(mean(h^2) + eps)) * (1 + w)),   packed = MXINT8(n)
//
// T is the residual stream's type: h is rounded once, and the norm is that of the stored h, as where the
// steps are calls of their own; n is rounded to bf16 as the decoder's separate norm writes it, so that packed
// is what a quantisation of those rows makes.
#include <algorithm>

#include "../../include/qwen_mlp.h"
#include "qmlp_internal.h"
#include "qmlp_mx8.h"

namespace qmlp {

constexpr int kNoAdd = -1;  // RT: nothing is added

// Rounds v to the residual stream's type, as the sum that is stored.
template <int RT>
__device__ __forceinline__ float stream_round(float v) {
  if constexpr (RT == QMLP_X_BF16) return bf16_to_f32(f32_to_bf16(v));
  return v;
}

template <int T>
__device__ __forceinline__ void store16(uint8_t* p, const float (&f)[16]) {  // of type T, which holds them exactly
  if constexpr (T == QMLP_X_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) *(f32x4*)(p + 16 * i) = f32x4{f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]};
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = (__float_as_uint(f[8 * i + 2 * j]) >> 16) | (__float_as_uint(f[8 * i + 2 * j + 1]) & 0xffff0000u);
      *(u32x4*)(p + 16 * i) = v;
    }
  }
}

// One workgroup a row, 16 values ("a chunk") a thread; REGS: the row's chunks are no more than the threads.
// Otherwise the sums are read again from where they were stored (by the same thread).
template <int XT, int RT, bool REGS>
__global__ __launch_bounds__(1024) void add_norm_kernel(AddNorm a) {
  __shared__ float s_sum[16];
  constexpr int kX = XT == QMLP_X_F32 ? 64 : 32, kR = RT == QMLP_X_F32 ? 64 : 32;  // bytes of a chunk
  const int m = blockIdx.x, tid = threadIdx.x, nch = a.cols / 16, nsb = mx_ksb(a.cols);
  const uint8_t* xr = a.x + (size_t)m * a.x_bytes;
  const uint8_t* rr = RT == kNoAdd ? nullptr : a.r + (size_t)m * a.r_bytes;
  uint8_t* hr = RT == kNoAdd ? nullptr : a.h + (size_t)m * a.h_bytes;
  auto sums = [&](int c, float (&f)[16]) {
    MxWords<XT> x[2];
    mx8_load<XT>(xr + (size_t)c * kX, x);
    mx8_floats<XT>(x, f);
    if constexpr (RT != kNoAdd) {
      constexpr int T = RT == kNoAdd ? 0 : RT;
      MxWords<T> r[2];
      mx8_load<T>(rr + (size_t)c * kR, r);
      float g[16];
      mx8_floats<T>(r, g);
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = stream_round<RT>(f[i] + g[i]);
      store16<T>(hr + (size_t)c * kR, f);
    }
  };
  auto again = [&](int c, float (&f)[16]) {  // a chunk whose sums were stored
    if constexpr (RT == kNoAdd) {
      sums(c, f);
    } else {
      constexpr int T = RT == kNoAdd ? 0 : RT;
      MxWords<T> h[2];
      mx8_load<T>(hr + (size_t)c * kR, h);
      mx8_floats<T>(h, f);
    }
  };
  float f[16], ss = 0.f;
  auto square = [&]() {
#pragma unroll
    for (int i = 0; i < 16; ++i) ss = fmaf(f[i], f[i], ss);
  };
  MxWords<0> w[2];
  if constexpr (REGS) {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = 0.f;
    w[0] = w[1] = MxWords<0>{};
    if (tid < nch) {
      mx8_load<0>((const uint8_t*)a.w + tid * 32, w);
      sums(tid, f);
    }
    square();
  } else {
    for (int c = tid; c < nch; c += blockDim.x) {
      sums(c, f);
      square();
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
  if ((tid & 63) == 0) s_sum[tid >> 6] = ss;
  __syncthreads();
  ss = 0.f;
  for (int i = 0; i < (int)blockDim.x / 64; ++i) ss += s_sum[i];
  const float rs = 1.0f / sqrtf(ss / (float)a.cols + a.eps);
  uint8_t* units = a.packed ? a.packed + (size_t)(m / kMxRows) * nsb * kMx8Unit : nullptr;
  // chunk c, up to the unit's end (zeros behind the row: the padding); all lanes of a wave take part
  auto emit = [&](int c) {
    float g[16];
    mx8_floats<0>(w, g);
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = c < nch ? bf16_to_f32(f32_to_bf16(f[i] * rs * (1.0f + g[i]))) : 0.f;
    if (a.n && c < nch) store16<QMLP_X_BF16>((uint8_t*)(a.n + (size_t)m * a.cols + (size_t)c * 16), f);
    if (units) {
      uint32_t top = abs_max16(f);
      top = max(top, (uint32_t)__shfl_xor((int)top, 1));
      const uint32_t s = mx8_scale_byte(top);
      if (c < nsb * 16) {
        uint8_t* unit = units + (size_t)(c / 16) * kMx8Unit;
        const int row = m % kMxRows, kb = (c / 2) % 8;
        *(i32x4*)(unit + mx8_at(row, kb, c & 1)) = mx8_group(f, s);
        if ((c & 1) == 0) unit[mx8_scale_at(row, kb)] = (uint8_t)s;
      }
    }
  };
  if constexpr (REGS) {
    emit(tid);
  } else {
    for (int c0 = 0; c0 < nsb * 16; c0 += blockDim.x) {
      const int c = min(c0 + tid, nch - 1);
      mx8_load<0>((const uint8_t*)a.w + (size_t)c * 32, w);
      again(c, f);
      emit(c0 + tid);
    }
  }
}

template <int XT, int RT>
static int launch_norm(const AddNorm& a, hipStream_t s) {
  const int chunks = mx_ksb(a.cols) * 16, threads = std::min(1024, (chunks + 63) / 64 * 64);
  auto kern = chunks <= 1024 ? add_norm_kernel<XT, RT, true> : add_norm_kernel<XT, RT, false>;
  hipLaunchKernelGGL(kern, dim3(a.rows), dim3(threads), 0, s, a);
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
