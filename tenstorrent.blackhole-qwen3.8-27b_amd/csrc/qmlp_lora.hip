// qmlp_lora.hip -- low-rank adapters of many requests at once (layouts: qmlp_lora.h).
//
// Two launches: lora_down_kernel makes t = A_a x of every token, lora_up_kernel adds s_a B_a t to the base.
// Both go by tiles of tokens that share an adapter, so that an adapter is read once a tile.
#include <algorithm>
#include <atomic>

#include "qmlp_lora.h"

namespace qmlp {

// ---------------------------------------------------------------- the plan
//
// One workgroup: counts the tokens of each adapter (ids outside [0, adapters) count as none), lays the
// groups out one after the other, those without an adapter last, and writes tiles and order.  The order inside a
// group is not fixed; no result depends on it.  Once a batch: its tokens' plan serves every projection of
// every layer.
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void lora_plan_kernel(const int* __restrict__ ids, int M, int adapters,
                                                                int* __restrict__ plan, int max_tiles) {
  constexpr int kSlots = 2 * kPlanThreads;  // adapters + 1 of them at most
  static_assert(kLoraMaxAdapters < kSlots);
  __shared__ int s_count[kSlots], s_scan[kPlanThreads], s_tiles[kPlanThreads];
  const int tid = threadIdx.x, T = lora_tile(M);
  for (int i = tid; i < kSlots; i += kPlanThreads) s_count[i] = 0;
  __syncthreads();
  auto slot = [&](int m) {
    const int id = ids[m];
    return id >= 0 && id < adapters ? id : adapters;
  };
  for (int m = tid; m < M; m += kPlanThreads) atomicAdd(&s_count[slot(m)], 1);
  __syncthreads();
  // two slots a thread: prefix sums of rows and tiles
  const int c0 = s_count[2 * tid], c1 = s_count[2 * tid + 1];
  const int t0 = (c0 + T - 1) / T, t1 = (c1 + T - 1) / T;
  s_scan[tid] = c0 + c1;
  s_tiles[tid] = t0 + t1;
  __syncthreads();
  for (int d = 1; d < kPlanThreads; d <<= 1) {
    const int a = tid >= d ? s_scan[tid - d] : 0, b = tid >= d ? s_tiles[tid - d] : 0;
    __syncthreads();
    s_scan[tid] += a;
    s_tiles[tid] += b;
    __syncthreads();
  }
  const int rows = s_scan[tid] - c0 - c1, tiles = s_tiles[tid] - t0 - t1;
  int* tile = plan + 4;
  auto write = [&](int which, int first_row, int count, int first_tile) {
    for (int i = 0; i * T < count; ++i) {
      int* p = tile + 4 * (first_tile + i);
      p[0] = which < adapters ? which : -1;
      p[1] = first_row + i * T;
      p[2] = min(T, count - i * T);
      p[3] = 0;
    }
  };
  write(2 * tid, rows, c0, tiles);
  write(2 * tid + 1, rows + c0, c1, tiles + t0);
  if (tid == kPlanThreads - 1) {
    plan[0] = kLoraMagic;
    plan[1] = M;
    plan[2] = adapters;
    plan[3] = s_tiles[tid];
  }
  __syncthreads();
  s_count[2 * tid] = rows;  // now the next place of each group
  s_count[2 * tid + 1] = rows + c0;
  __syncthreads();
  int* order = tile + 4 * max_tiles;
  for (int m = tid; m < M; m += kPlanThreads) order[atomicAdd(&s_count[slot(m)], 1)] = m;
}

int launch_lora_plan(const int* ids, int M, int adapters, int* plan, hipStream_t s) {
  hipLaunchKernelGGL(lora_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, ids, M, adapters, plan,
                     lora_max_tiles(M, adapters));
  return check_launch("lora_plan_kernel");
}

struct LoraTile {
  int adapter, first, rows;
};
// Tile t of a plan; rows 0 where there is none, or where the plan is not one for these sizes.
__device__ __forceinline__ LoraTile lora_tile_of(const int* plan, int t, int M, int adapters) {
  if (plan[0] != kLoraMagic || plan[1] != M || plan[2] != adapters || t >= plan[3]) return LoraTile{-1, 0, 0};
  const int* p = plan + 4 + 4 * t;
  return LoraTile{p[0], p[1], p[2]};
}

template <bool F16>
__device__ __forceinline__ f32x4 lora_product(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}

// ---------------------------------------------------------------- A x
//
// One workgroup of 8 waves per (tile, K piece); the waves share the piece's K-steps of 32 out in turn and add
// their sums up in a fixed order through LDS.  TU: units of 16 tokens of a tile; RU: rank units at most.
constexpr int kDownWaves = 8;
template <bool F16, int TU, int RU>
__global__ __launch_bounds__(kDownWaves * 64, 1) void lora_down_kernel(LoraArgs p, int max_tiles, int ranks) {
  extern __shared__ __align__(16) float s_sum[];  // [kDownWaves / 2][TU][RU][64 lanes][4]
  const LoraTile t = lora_tile_of(p.plan, blockIdx.x, p.M, p.adapters);
  if (t.adapter < 0 || t.rows == 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int* meta = p.stack.meta + 4 * t.adapter;
  const int rank = meta[0], steps = p.K / 32, pieces = gridDim.y;
  const int ru = min((rank + 15) / 16, RU), tu = (t.rows + 15) / 16;
  const int s0 = blockIdx.y * steps / pieces, s1 = (blockIdx.y + 1) * steps / pieces;
  const uint8_t* a = p.stack.a + ((size_t)meta[1] * steps * 64 + lane) * 16;
  const int* order = p.plan + 4 + 4 * max_tiles + t.first;
  const uint8_t* x[TU];
#pragma unroll
  for (int u = 0; u < TU; ++u)  // rows behind the tile's last one read it again
    x[u] = p.x + (size_t)order[min(u * 16 + (lane & 15), t.rows - 1)] * p.x_bytes + (lane >> 4) * 16;
  bool mine[RU];  // ranks that the adapter has
#pragma unroll
  for (int r = 0; r < RU; ++r) mine[r] = r * 16 + (lane & 15) < rank;
  f32x4 acc[TU][RU];
#pragma unroll
  for (int u = 0; u < TU; ++u)
#pragma unroll
    for (int r = 0; r < RU; ++r) acc[u][r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int s = s0 + wave; s < s1; s += kDownWaves) {
    u32x4 av[RU], xv[TU];
#pragma unroll
    for (int r = 0; r < RU; ++r)
      av[r] = mine[r] ? *(const u32x4*)(a + ((size_t)r * steps + s) * 1024) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int u = 0; u < TU; ++u)
      if (u < tu) xv[u] = *(const u32x4*)(x[u] + (size_t)s * 64);
#pragma unroll
    for (int u = 0; u < TU; ++u)
      if (u < tu) {
#pragma unroll
        for (int r = 0; r < RU; ++r)
          if (r < ru) acc[u][r] = lora_product<F16>(av[r], xv[u], acc[u][r]);
      }
  }
#pragma unroll
  for (int half = kDownWaves / 2; half > 0; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
      f32x4* at = (f32x4*)s_sum + (size_t)(wave - half) * TU * RU * 64 + lane;
#pragma unroll
      for (int u = 0; u < TU; ++u)
#pragma unroll
        for (int r = 0; r < RU; ++r) at[(u * RU + r) * 64] = acc[u][r];
    }
    __syncthreads();
    if (wave < half) {
      const f32x4* at = (const f32x4*)s_sum + (size_t)wave * TU * RU * 64 + lane;
#pragma unroll
      for (int u = 0; u < TU; ++u)
#pragma unroll
        for (int r = 0; r < RU; ++r) acc[u][r] += at[(u * RU + r) * 64];
    }
    __syncthreads();
  }
  if (wave != 0) return;
  // lane: token lane % 16 of a unit, ranks 16 r + 4 (lane / 16)..
#pragma unroll
  for (int u = 0; u < TU; ++u) {
    const int row = u * 16 + (lane & 15);
    if (row >= t.rows) continue;
    float* o = p.parts + ((size_t)blockIdx.y * p.M + t.first + row) * ranks + 4 * (lane >> 4);
#pragma unroll
    for (int r = 0; r < RU; ++r)
      if (r < ru) *(f32x4*)(o + 16 * r) = acc[u][r];
  }
}

// ---------------------------------------------------------------- base + s B t
//
// One workgroup of 4 waves per (tile, run of feature blocks).  It adds the pieces of t up in order, scales them
// and splits each fp32 sum into three 16-bit numbers whose sum it is but for 2^-24 of it (bf16), or of the
// token's largest (fp16: over a power of two that brings the largest near the type's), so the products keep
// fp32's accuracy; they are laid out in LDS as the products' operands.  An operand of 32 holds 16 ranks twice: the
// first parts beside the second ones; a second product adds the third parts.
constexpr int kUpWaves = 4;
template <bool F16>
__device__ __forceinline__ uint32_t lora_round(float v) {  // to the adapters' type
  if constexpr (F16) return f32_to_f16_bits(v);
  return f32_to_bf16(v);
}
template <bool F16>
__device__ __forceinline__ float lora_value(uint32_t b) {
  if constexpr (F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)b);
  return bf16_to_f32((uint16_t)b);
}

template <bool F16, int TU>
__global__ __launch_bounds__(kUpWaves * 64) void lora_up_kernel(LoraArgs p, int max_tiles, int ranks, int pieces,
                                                               int blocks_each) {
  extern __shared__ __align__(16) uint8_t s_t[];  // [rank unit][token unit][2][lane][8] 16-bit numbers
  __shared__ float s_scale[TU * 16];               // fp16: what a token's sums are multiplied by
  const LoraTile t = lora_tile_of(p.plan, blockIdx.x, p.M, p.adapters);
  if (t.rows == 0 || (t.adapter < 0 && p.base == p.out)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int blocks = (p.N + 63) / 64;
  const int b0 = blockIdx.y * blocks_each, b1 = min(blocks, b0 + blocks_each);
  const int* order = p.plan + 4 + 4 * max_tiles + t.first;
  int rank = 0, first = 0;
  float s = 0.f;
  if (t.adapter >= 0) {
    const int* meta = p.stack.meta + 4 * t.adapter;
    rank = min(meta[0], ranks);
    first = meta[1];
    s = __int_as_float(meta[2]);
  }
  const int ru = (rank + 15) / 16, tu = (t.rows + 15) / 16;
  if (ru) {
    // a thread: 8 ranks of a token
    const int items = tu * 16 * ru * 2;
    auto sum8 = [&](int row, int r8, float (&v)[8]) {
      f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
      const float* at = p.parts + (size_t)(t.first + row) * ranks + r8 * 8;
      for (int q = 0; q < pieces; ++q, at += (size_t)p.M * ranks) {
        lo += *(const f32x4*)at;
        hi += *(const f32x4*)(at + 4);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = lo[i] * s;
        v[4 + i] = hi[i] * s;
      }
    };
    if constexpr (F16) {
      // the token's power of two: 2 ru items of a row are neighbours in neither wave nor time, so one thread a row
      for (int row = tid; row < TU * 16; row += kUpWaves * 64) {
        float m = 0.f;
        if (row < t.rows)
          for (int r8 = 0; r8 < 2 * ru; ++r8) {
            float v[8];
            sum8(row, r8, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
          }
        const int e = (int)(__float_as_uint(m) >> 23);  // the largest becomes one of [2^14, 2^15)
        s_scale[row] = __uint_as_float((uint32_t)(min(max(e, 16), 254) - 14) << 23);
      }
      __syncthreads();
    }
    for (int item = tid; item < items; item += kUpWaves * 64) {
      const int row = item / (2 * ru), r8 = item % (2 * ru);
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
      if (row < t.rows) sum8(row, r8, v);
      float inv = 1.f;
      if constexpr (F16) inv = 1.0f / s_scale[row];  // a power of two: exact
      u32x4 part[3];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float rest = v[i] * inv;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const uint32_t b = lora_round<F16>(rest);
          rest = __builtin_isfinite(rest) ? rest - lora_value<F16>(b) : 0.f;
          part[k][i / 2] = i % 2 ? part[k][i / 2] | b << 16 : b;
        }
      }
      // lane of an operand: token row % 16, K 8 (lane / 16)..: ranks 0..15, then again
      uint8_t* at = s_t + ((size_t)(r8 / 2) * TU + row / 16) * 2048 + ((r8 & 1) * 16 + row % 16) * 16;
      *(u32x4*)at = part[0];
      *(u32x4*)(at + 512) = part[1];
      *(u32x4*)(at + 1024) = part[2];
      *(u32x4*)(at + 1536) = u32x4{0u, 0u, 0u, 0u};
    }
    __syncthreads();
  }
  const bool whole = p.N % 8 == 0;  // rows that vector accesses of 8 features divide
  const size_t bblock = (size_t)ru * 2048;
  const uint8_t* bmat = p.stack.b + (size_t)first * ((size_t)blocks * 2048) + (lane & 31) * 16;
  const int g = lane >> 4;
  for (int b = b0 + wave; b < b1; b += kUpWaves) {
    f32x4 acc[TU][4];
#pragma unroll
    for (int u = 0; u < TU; ++u)
#pragma unroll
      for (int f = 0; f < 4; ++f) acc[u][f] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int r = 0; r < ru; ++r) {
      u32x4 w[4];
      const bool mine = r * 16 + ((lane >> 4) & 1) * 8 < rank;
#pragma unroll
      for (int f = 0; f < 4; ++f)
        w[f] = mine ? *(const u32x4*)(bmat + b * bblock + (r * 4 + f) * 512) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int u = 0; u < TU; ++u)
        if (u < tu) {
          const uint8_t* at = s_t + ((size_t)r * TU + u) * 2048 + lane * 16;
          const u32x4 t01 = *(const u32x4*)at, t2 = *(const u32x4*)(at + 1024);
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            acc[u][f] = lora_product<F16>(w[f], t2, acc[u][f]);
            acc[u][f] = lora_product<F16>(w[f], t01, acc[u][f]);
          }
        }
    }
    // lane: token lane % 16 of a unit, features 64 b + 16 g..
#pragma unroll
    for (int u = 0; u < TU; ++u) {
      const int row = u * 16 + (lane & 15);
      if (row >= t.rows) continue;
      float m = 1.f;
      if constexpr (F16)
        if (ru) m = s_scale[row];
      const size_t at0 = (size_t)order[row] * p.N;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int n = b * 64 + g * 16 + h * 8;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = acc[u][2 * h + i / 4][i % 4] * m;
        if (whole && n < p.N) {
          const size_t at = at0 + n;
          if (p.base) {
            if (p.base_f32) {
              const f32x4 lo = *(const f32x4*)((const float*)p.base + at), hi = *(const f32x4*)((const float*)p.base + at + 4);
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] += i < 4 ? lo[i] : hi[i - 4];
            } else {
              const u32x4 w = *(const u32x4*)((const uint16_t*)p.base + at);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                v[2 * i] += __uint_as_float(w[i] << 16);
                v[2 * i + 1] += __uint_as_float(w[i] & 0xffff0000u);
              }
            }
          }
          if (p.out_f32) {
            *(f32x4*)((float*)p.out + at) = f32x4{v[0], v[1], v[2], v[3]};
            *(f32x4*)((float*)p.out + at + 4) = f32x4{v[4], v[5], v[6], v[7]};
          } else {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = (uint32_t)f32_to_bf16(v[2 * i]) | (uint32_t)f32_to_bf16(v[2 * i + 1]) << 16;
            *(u32x4*)((uint16_t*)p.out + at) = w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (n + i >= p.N) continue;
            const size_t at = at0 + n + i;
            if (p.base)
              v[i] += p.base_f32 ? ((const float*)p.base)[at] : bf16_to_f32(((const uint16_t*)p.base)[at]);
            if (p.out_f32)
              ((float*)p.out)[at] = v[i];
            else
              ((uint16_t*)p.out)[at] = f32_to_bf16(v[i]);
          }
        }
      }
    }
  }
}

// ---------------------------------------------------------------- launches

static int up_div(int a, int b) { return (a + b - 1) / b; }

// Enough workgroups for the card at two K-steps a wave or more, as far as the tiles alone are not: the most
// tiles that M tokens can make are counted as half of them, since an adapter's tokens share tiles as a rule.
int lora_pieces(int M, int K, int adapters, int num_cus) {
  const int tiles = std::max(1, lora_max_tiles(M, adapters) / 2);
  return std::max(1, std::min({kLoraMaxPieces, up_div(K / 32, 2 * kDownWaves),
                               up_div(std::min(num_cus, kMaxWorkgroups), tiles)}));
}

static int padded_rank(int rank) { return (rank + 15) / 16 * 16; }

// The most that pieces x M can be, whatever the adapters and the card: there are M / 128 or more of lora_pieces'
// tiles (of M / 64 + 2 or more, halved), hence at most 512 / (M / 128) + 1 pieces.
size_t lora_parts_bytes(int M, int K, int max_rank) {
  const int most = std::max(1, std::min(kLoraMaxPieces, up_div(K / 32, 2 * kDownWaves)));
  const size_t rows = std::min((size_t)most * M, (size_t)kMaxWorkgroups * 128 + M);
  return align256(rows * padded_rank(max_rank) * 4);
}

template <bool F16, int TU, int RU>
static int launch_down(const LoraArgs& a, int max_tiles, int pieces, hipStream_t s) {
  constexpr size_t lds = (size_t)kDownWaves / 2 * TU * RU * 64 * 16;
  auto kern = lora_down_kernel<F16, TU, RU>;
  if constexpr (lds > 65536) {
    static std::atomic<uint64_t> raised{0};
    if (int rc = raise_lds_once((const void*)kern, (int)lds, raised)) return rc;
  }
  hipLaunchKernelGGL(kern, dim3(max_tiles, pieces), dim3(kDownWaves * 64), lds, s, a, max_tiles,
                     padded_rank(a.max_rank));
  return check_launch("lora_down_kernel");
}

template <bool F16, int TU>
static int launch_tokens(const LoraArgs& a, int num_cus, hipStream_t s) {
  const int max_tiles = lora_max_tiles(a.M, a.adapters), pieces = lora_pieces(a.M, a.K, a.adapters, num_cus);
  const int units = padded_rank(a.max_rank) / 16;
  const int rc = units <= 1   ? launch_down<F16, TU, 1>(a, max_tiles, pieces, s)
                 : units <= 2 ? launch_down<F16, TU, 2>(a, max_tiles, pieces, s)
                 : units <= 4 ? launch_down<F16, TU, 4>(a, max_tiles, pieces, s)
                              : launch_down<F16, TU, 8>(a, max_tiles, pieces, s);
  if (rc) return rc;
  const int blocks = up_div(a.N, 64), tiles = std::max(1, max_tiles / 2);
  const int runs = std::max(1, std::min(up_div(blocks, kUpWaves), up_div(4 * num_cus, tiles)));
  const int each = up_div(blocks, runs);
  const size_t lds = (size_t)units * TU * 2048;
  auto up = lora_up_kernel<F16, TU>;
  if constexpr (TU > 1) {  // 64 KB at the largest rank, besides the scales
    static std::atomic<uint64_t> raised{0};
    if (int rc = raise_lds_once((const void*)up, kLoraMaxRank / 16 * TU * 2048, raised)) return rc;
  }
  hipLaunchKernelGGL(up, dim3(max_tiles, up_div(blocks, each)), dim3(kUpWaves * 64), lds, s, a,
                     max_tiles, padded_rank(a.max_rank), pieces, each);
  return check_launch("lora_up_kernel");
}

int launch_lora(const LoraArgs& a, int num_cus, hipStream_t s) {
  if (lora_tile(a.M) == 16) return a.f16 ? launch_tokens<true, 1>(a, num_cus, s) : launch_tokens<false, 1>(a, num_cus, s);
  return a.f16 ? launch_tokens<true, 4>(a, num_cus, s) : launch_tokens<false, 4>(a, num_cus, s);
}

}  // namespace qmlp
