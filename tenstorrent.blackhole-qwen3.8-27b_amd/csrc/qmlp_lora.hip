// qmlp_lora.hip -- low-rank adapters of many requests at once (layouts: qmlp_lora.h).
//
// Two launches: lora_down_kernel makes t = A_a x of every token, lora_up_kernel adds s_a B_a t to the base; or one,
// where A and a few tokens' rows are little to read again.  Both go by tiles of tokens that share an adapter.
#include <algorithm>
#include <atomic>

#include "qmlp_lora.h"
#include "qmlp_mx.h"

namespace qmlp {

// ---------------------------------------------------------------- the plan
//
// One workgroup: counts the tokens of each adapter (ids outside [0, adapters) count as none), lays the
// groups out one after the other, those without an adapter last, and writes tiles and order.  The order inside a
// group is not fixed; no result depends on it.  Once a batch: its tokens' plan serves every projection of
// every layer.  Bound by its steps' latencies; captured: 4.1-4.9 us up to 512 tokens, 5.1-6.0 for 2048, and for 65536 36 in
// any order of eight adapters, 40 of one adapter, 56 in any order of 1024.
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void lora_plan_kernel(const int* __restrict__ ids, int M, int adapters,
                                                                int* __restrict__ plan, int max_tiles) {
  constexpr int kSlots = 2 * kPlanThreads;  // adapters + 1 of them at most
  static_assert(kLoraMaxAdapters < kSlots);
  __shared__ int s_count[kSlots], s_scan[kPlanThreads], s_tiles[kPlanThreads], s_wave[2][kPlanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, T = lora_tile(M);
  for (int i = tid; i < kSlots; i += kPlanThreads) s_count[i] = 0;
  __syncthreads();
  auto slot = [&](int m) {
    const int id = ids[m];
    return id >= 0 && id < adapters ? id : adapters;
  };
  // The next place of token m's group.  Requests' tokens come in runs, and a wave whose tokens share a group takes
  // their places at once: with places taken one by one and a group's tiles written by one thread 65536 tokens of one
  // adapter took 193 us and 2048 11, for 40 and 5.1.
  auto take = [&](int m) {
    const int k = slot(m), first = __builtin_amdgcn_readfirstlane(k);
    if (!__all(k == first)) return atomicAdd(&s_count[k], 1);
    const uint64_t active = __ballot(1);
    const int before = __builtin_popcountll(active & ((1ull << lane) - 1));
    int at = 0;
    if (before == 0) at = atomicAdd(&s_count[first], __builtin_popcountll(active));
    return __builtin_amdgcn_readfirstlane(at) + before;
  };
  for (int m = tid; m < M; m += kPlanThreads) take(m);
  __syncthreads();
  // two slots a thread: prefix sums of rows and tiles
  const int c0 = s_count[2 * tid], c1 = s_count[2 * tid + 1];
  const int t0 = (c0 + T - 1) / T, t1 = (c1 + T - 1) / T;
  int sum_rows = c0 + c1, sum_tiles = t0 + t1;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int a = __shfl_up(sum_rows, d), b = __shfl_up(sum_tiles, d);
    if (lane >= d) {
      sum_rows += a;
      sum_tiles += b;
    }
  }
  if (lane == 63) {
    s_wave[0][tid / 64] = sum_rows;
    s_wave[1][tid / 64] = sum_tiles;
  }
  __syncthreads();
  for (int w = 0; w < tid / 64; ++w) {
    sum_rows += s_wave[0][w];
    sum_tiles += s_wave[1][w];
  }
  s_scan[tid] = sum_rows;
  s_tiles[tid] = sum_tiles;
  __syncthreads();
  const int rows = s_scan[tid] - c0 - c1;
  int* tile = plan + 4;
  const int tiles = s_tiles[kPlanThreads - 1];
  for (int t = tid; t < tiles; t += kPlanThreads) {
    int lo = 0, hi = adapters / 2;  // the pair of slots that tile t belongs to
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (s_tiles[mid] > t) hi = mid; else lo = mid + 1;
    }
    int which = 2 * lo, count = s_count[which], next = s_count[which + 1];
    const int own = (count + T - 1) / T;
    int i = t - (s_tiles[lo] - own - (next + T - 1) / T), row = s_scan[lo] - count - next;
    if (i >= own) {
      i -= own;
      row += count;
      count = next;
      ++which;
    }
    *(int4*)(tile + 4 * t) = make_int4(which < adapters ? which : -1, row + i * T, min(T, count - i * T), 0);
  }
  if (tid == kPlanThreads - 1) {
    plan[0] = kLoraMagic;
    plan[1] = M;
    plan[2] = adapters;
    plan[3] = tiles;
  }
  __syncthreads();
  s_count[2 * tid] = rows;  // now the next place of each group
  s_count[2 * tid + 1] = rows + c0;
  __syncthreads();
  int* order = tile + 4 * max_tiles;
  for (int m = tid; m < M; m += kPlanThreads) order[take(m)] = m;
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
  typedef int i32x4_t __attribute__((ext_vector_type(4)));
  const i32x4_t head = *(const i32x4_t*)plan, p = *(const i32x4_t*)(plan + 4 + 4 * t);  // on their way together
  const bool ok = (head.x == kLoraMagic) & (head.y == M) & (head.z == adapters) & (t < head.w);
  return LoraTile{ok ? p.x : -1, ok ? p.y : 0, ok ? p.z : 0};
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
// One workgroup of 8 (few tokens: 16) waves per (K piece, tile): with eight pieces each XCD reads one of them of
// every adapter, which its L2 holds.  The waves share the piece's K-steps of 32 out in turn, two neighbouring ones
// (a line of a 16-bit row) at a time, and add their sums up in a fixed order through LDS.  Rows of x come in by
// whole lines, 8 lanes to a row, and turn through LDS into operands: read as the operands lie, one row a lane,
// every lane of a load is an access of its own, and those bounded the kernel (27000 of a CU for 2048 x 17408).  It
// takes 22 us there with rank 64: 71 MB of x and, from the L2s, 143 MB of A, which each 32 tokens read again,
// 9.7 TB/s into the CUs.  Loads of two and three steps under way instead of one change nothing (23.2 and 23.1 us), nor
// do tiles of 64 tokens, which read A half as often (both launches 33.8 us for 32.6 there, 62.7 for 68.0 at 4096
// tokens, 18.3 for 16.9 at 777 and rank 16).
// TU: units of 16 tokens of a tile; RU: rank units at most.
template <int TU, int RU>
constexpr int kDownWaves = TU == 1 && RU <= 4 ? 16 : 8;  // 128 ranks take the registers of two waves
template <int TU, int RU>
constexpr size_t kDownLds = kDownWaves<TU, RU> * TU * (RU > 4 ? RU * 512 : 2048);  // turning, then the waves' sums

// The sums of K-steps s0..s1 of one tile, in wave 0 of kDownWaves: lane: token lane % 16 of a unit, ranks 16 r + 4
// (lane / 16)..
template <bool F16, int TU, int RU>
__device__ __forceinline__ void lora_down_tile(const LoraArgs& p, const LoraTile& t, const int* order, int rank, int first,
                                               int s0, int s1, uint8_t* s_mem, f32x4 (&acc)[TU][RU]) {
  constexpr int kWaves = kDownWaves<TU, RU>, kLoads = 2 * TU;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint8_t* x[kLoads];  // load i: rows 8 i + lane / 8, 16 bytes at 16 (lane % 8) of the two steps' line
  bool row_in[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = 8 * i + (lane >> 3);
    row_in[i] = row < t.rows;
    x[i] = p.x + (size_t)order[min(row, t.rows - 1)] * p.x_bytes + (lane & 7) * 16;
  }
  const int steps = p.K / 32, ru = (rank + 15) / 16, tu = (t.rows + 15) / 16;
  const uint8_t* a = p.stack.a + ((size_t)first * steps * 64 + lane) * 16;
  bool mine[RU];  // ranks that the adapter has
#pragma unroll
  for (int r = 0; r < RU; ++r) mine[r] = r * 16 + (lane & 15) < rank;
  u32x4 av[2][RU], xv[kLoads];
  auto load = [&](int s) {  // a step behind the piece multiplies zeros by zeros
    const bool second = s + 1 < s1;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      xv[i] = row_in[i] && (second || (lane & 4) == 0) ? *(const u32x4*)(x[i] + (size_t)s * 64) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int d = 0; d < 2; ++d)
#pragma unroll
      for (int r = 0; r < RU; ++r)
        av[d][r] = mine[r] && (d == 0 || second) ? *(const u32x4*)(a + ((size_t)r * steps + s + d) * 1024)
                                                 : u32x4{0u, 0u, 0u, 0u};
  };
#pragma unroll
  for (int u = 0; u < TU; ++u)
#pragma unroll
    for (int r = 0; r < RU; ++r) acc[u][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint8_t* turn = s_mem + wave * TU * 2048;  // a row's 8 pieces of 16 bytes, piece c at c ^ (row % 8)
  auto turn_fence = [] {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  if (s0 + 2 * wave < s1) load(s0 + 2 * wave);
  for (int s = s0 + 2 * wave; s < s1; s += 2 * kWaves) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = 8 * i + (lane >> 3);
      *(u32x4*)(turn + row * 128 + (((lane & 7) ^ (row & 7)) * 16)) = xv[i];
    }
    u32x4 w[2][RU];
#pragma unroll
    for (int d = 0; d < 2; ++d)
#pragma unroll
      for (int r = 0; r < RU; ++r) w[d][r] = av[d][r];
    if (s + 2 * kWaves < s1) load(s + 2 * kWaves);
    turn_fence();
#pragma unroll
    for (int d = 0; d < 2; ++d)
#pragma unroll
      for (int u = 0; u < TU; ++u)
        if (u < tu) {
          const int row = u * 16 + (lane & 15);
          const u32x4 v = *(const u32x4*)(turn + row * 128 + (((d * 4 + (lane >> 4)) ^ (row & 7)) * 16));
#pragma unroll
          for (int r = 0; r < RU; ++r)
            if (r < ru) acc[u][r] = lora_product<F16>(w[d][r], v, acc[u][r]);
        }
    turn_fence();
  }
  __syncthreads();
  f32x4* s_sum = (f32x4*)s_mem;  // [kWaves / 2][TU][RU][64 lanes]
#pragma unroll
  for (int half = kWaves / 2; half > 0; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
      f32x4* at = s_sum + (size_t)(wave - half) * TU * RU * 64 + lane;
#pragma unroll
      for (int u = 0; u < TU; ++u)
#pragma unroll
        for (int r = 0; r < RU; ++r) at[(u * RU + r) * 64] = acc[u][r];
    }
    __syncthreads();
    if (wave < half) {
      const f32x4* at = s_sum + (size_t)wave * TU * RU * 64 + lane;
#pragma unroll
      for (int u = 0; u < TU; ++u)
#pragma unroll
        for (int r = 0; r < RU; ++r) acc[u][r] += at[(u * RU + r) * 64];
    }
    __syncthreads();
  }
}

template <bool F16, int TU, int RU>
__global__ __launch_bounds__((kDownWaves<TU, RU> * 64), 1) void lora_down_kernel(LoraArgs p, int max_tiles, int ranks) {
  extern __shared__ __align__(16) uint8_t s_mem[];
  const LoraTile t = lora_tile_of(p.plan, blockIdx.y, p.M, p.adapters);
  if (t.adapter < 0 || t.rows == 0) return;
  const int* meta = p.stack.meta + 4 * t.adapter;
  const int rank = min(meta[0], ranks), steps = p.K / 32, pieces = gridDim.x;
  f32x4 acc[TU][RU];
  lora_down_tile<F16, TU, RU>(p, t, p.plan + 4 + 4 * max_tiles + t.first, rank, meta[1], blockIdx.x * steps / pieces,
                              (blockIdx.x + 1) * steps / pieces, s_mem, acc);
  const int lane = threadIdx.x;
  if (lane >= 64) return;
#pragma unroll
  for (int u = 0; u < TU; ++u) {
    const int row = u * 16 + (lane & 15);
    if (row >= t.rows) continue;
    float* o = p.parts + ((size_t)blockIdx.x * p.M + t.first + row) * ranks + 4 * (lane >> 4);
#pragma unroll
    for (int r = 0; r < RU; ++r)
      if (r * 16 < rank) *(f32x4*)(o + 16 * r) = acc[u][r];
  }
}

// ---------------------------------------------------------------- base + s B t
//
// One workgroup of 8 waves per (16 tokens of a tile, run of feature blocks).  It adds the pieces of t up, scales
// them and splits each fp32 sum into three 16-bit numbers whose sum it is but for 2^-24 of it (bf16), or of the
// token's largest (fp16: over a power of two that brings the largest near the type's), so the products keep
// fp32's accuracy; they are laid out in LDS as the products' operands, 32 ranks' parts of one order each.  Bound by
// memory: 16.7 us for 2048 tokens x 5120 with a bf16 base and rank 64, 70 MB read and written, 4.2 TB/s.
// DOWN: rank units that a workgroup (of up to 16 waves) makes t of by itself, 0 where lora_down_kernel did: one launch
// instead of two where that reads little.
constexpr int kUpParts = 3 * 1024;  // bytes of 32 ranks of 16 tokens
template <int DOWN>
constexpr int kUpWaves = DOWN ? kDownWaves<1, DOWN> : 8;
constexpr int kTurnRow = 68;  // floats of a token's row in LDS
// LDS: what makes t (DOWN), later the rows that turn; then the operands; then t in fp32.
template <int DOWN>
constexpr size_t kUpWork = kUpWaves<DOWN> * 16 * kTurnRow * 4;
template <int DOWN>
constexpr size_t lora_up_lds(int units) {
  return kUpWork<DOWN> + (size_t)(units + 1) / 2 * kUpParts + (size_t)units * 1024;
}
static_assert(kUpWork<8> >= kDownLds<1, 8> && kUpWork<4> >= kDownLds<1, 4>);
template <bool F16>
__device__ __forceinline__ uint32_t lora_round(float v) {  // to the adapters' type
  if constexpr (F16) return f32_to_f16_bits(v);
  return mx_bf16x2(v, 0.f) & 0xffffu;
}
template <bool F16>
__device__ __forceinline__ float lora_value(uint32_t b) {
  if constexpr (F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)b);
  return bf16_to_f32((uint16_t)b);
}

// Four ranks' sum over the pieces, in order.
__device__ __forceinline__ f32x4 lora_sum(const float* at, size_t piece, int pieces) {
  f32x4 v[kLoraMaxPieces];
#pragma unroll
  for (int q = 0; q < kLoraMaxPieces; ++q) v[q] = *(const f32x4*)(at + min(q, pieces - 1) * piece);
#pragma unroll
  for (int q = 1; q < kLoraMaxPieces; ++q)
    if (q < pieces) v[0] += v[q];
  return v[0];
}

// A block of 16 tokens x 64 features is finished by rows.  Rows of a multiple of 8 features (WHOLE): a lane takes 8
// neighbouring features of tokens lane / 8 and 8 more, so that 8 lanes touch 64 features of a token together.
// Others, which start anywhere: feature `lane` of all 16 tokens.  BASE: 0 none, 1 bf16, 2 fp32.
template <bool F16, bool WHOLE, int BASE, int DOWN>
__global__ __launch_bounds__(kUpWaves<DOWN> * 64) void lora_up_kernel(LoraArgs p, int max_tiles, int ranks, int pieces,
                                                                     int runs, int blocks_each, int tile_units) {
  constexpr int kWaves = kUpWaves<DOWN>, kThreads = kWaves * 64;
  extern __shared__ __align__(16) uint8_t s_work[];
  uint8_t* s_t = s_work + kUpWork<DOWN>;  // [32 ranks][3 parts][lane][8] 16-bit numbers, then t in fp32
  __shared__ float s_scale[16];           // fp16: what a token's sums are multiplied by
  // DOWN: a tile's runs share an XCD (block b runs on XCD b % 8), whose L2 keeps the A that they all read, where there
  // are tiles for every XCD
  const int b8 = blockIdx.x / 8, tiles = gridDim.x / runs;
  const bool grouped = DOWN && tiles % 8 == 0;
  const int run = !DOWN ? blockIdx.x / tiles : grouped ? b8 % runs : blockIdx.x % runs;
  const int tile = !DOWN ? blockIdx.x % tiles : grouped ? b8 / runs * 8 + blockIdx.x % 8 : blockIdx.x / runs;
  const int unit = tile % tile_units * 16;
  if (tile >= max_tiles * tile_units) return;
  LoraTile t = lora_tile_of(p.plan, tile / tile_units, p.M, p.adapters);
  t.first += unit;
  t.rows = min(16, t.rows - unit);
  if (t.rows <= 0 || (t.adapter < 0 && p.base == p.out)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int blocks = (p.N + 63) / 64;
  const int b0 = run * blocks_each, b1 = min(blocks, b0 + blocks_each);
  const int* order = p.plan + 4 + 4 * max_tiles + t.first;
  int rank = 0, first = 0, first_a = 0;
  float s = 0.f;
  if (t.adapter >= 0) {
    const int* meta = p.stack.meta + 4 * t.adapter;
    rank = min(meta[0], ranks);
    first_a = meta[1];
    s = __int_as_float(meta[2]);
    first = meta[3];
  }
  const int ru = (rank + 31) / 32;
  const size_t bblock = (size_t)ru * 4096;
  const uint8_t* bmat = p.stack.b + (size_t)first * ((size_t)blocks * 4096) + lane * 16;
  u32x4 w[4];
  auto load_w = [&](int b, int r) {
    const bool mine = r * 32 + (lane >> 4) * 8 < rank;
#pragma unroll
    for (int f = 0; f < 4; ++f)
      w[f] = mine ? *(const u32x4*)(bmat + b * bblock + (r * 4 + f) * 1024) : u32x4{0u, 0u, 0u, 0u};
  };
  // where this lane finishes: WHOLE: rows lane / 8 and 8 behind, features 8 (lane % 8)..
  const int half = WHOLE ? lane >> 3 : 0, n0 = WHOLE ? (lane & 7) * 8 : lane;
  const size_t at0 = (size_t)order[min(half, t.rows - 1)] * p.N, at1 = (size_t)order[min(WHOLE ? half + 8 : 0, t.rows - 1)] * p.N;
  u32x4 base[BASE == 1 && WHOLE ? 2 : 4];
  auto load_base = [&](int b) {
    const int n = b * 64 + n0;
    if (n >= p.N) return;
    if constexpr (BASE == 1 && WHOLE) {
      base[0] = *(const u32x4*)((const uint16_t*)p.base + at0 + n);
      base[1] = *(const u32x4*)((const uint16_t*)p.base + at1 + n);
    } else if constexpr (BASE == 2 && WHOLE) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        base[i] = *(const u32x4*)((const float*)p.base + (i < 2 ? at0 : at1) + n + i % 2 * 4);
    } else if constexpr (BASE != 0) {  // tokens behind the last one read it again
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const size_t at = (size_t)order[min(i, t.rows - 1)] * p.N + n;
        base[i / 4][i % 4] =
            BASE == 1 ? (uint32_t)((const uint16_t*)p.base)[at] << 16 : ((const uint32_t*)p.base)[at];
      }
    }
  };
  if (b0 + wave < b1) load_base(b0 + wave);
  if (b0 + wave < b1 && ru) load_w(b0 + wave, 0);
  if (ru) {
    const int row4 = (rank + 15) / 16 * 4;  // four ranks each
    f32x4* s_sum = (f32x4*)(s_t + (size_t)ru * kUpParts);
    if constexpr (DOWN) {
      f32x4 acc[1][DOWN];
      lora_down_tile<F16, 1, DOWN>(p, t, order, rank, first_a, 0, p.K / 32, s_work, acc);
      if (wave == 0 && (lane & 15) < t.rows) {
#pragma unroll
        for (int r = 0; r < DOWN; ++r)
          if (r * 16 < rank) s_sum[(lane & 15) * row4 + 4 * r + (lane >> 4)] = acc[0][r] * s;
      }
    } else {
      const float* at = p.parts + (size_t)t.first * ranks;
      for (int e = tid; e < t.rows * row4; e += kThreads)
        s_sum[e] = lora_sum(at + (size_t)(e / row4) * ranks + e % row4 * 4, (size_t)p.M * ranks, pieces) * s;
    }
    __syncthreads();
    if constexpr (F16) if (tid < 256) {
      const int row = tid / 16;
      float m = 0.f;
      if (row < t.rows)
        for (int r = tid % 16; r < row4; r += 16) {
          const f32x4 v = s_sum[row * row4 + r];
#pragma unroll
          for (int i = 0; i < 4; ++i) m = r * 4 + i < rank ? fmaxf(m, fabsf(v[i])) : m;
        }
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
      const int e = (int)(__float_as_uint(m) >> 23);  // the largest becomes one of [2^14, 2^15)
      s_scale[row] = __uint_as_float((uint32_t)(min(max(e, 16), 254) - 14) << 23);
    }
    if constexpr (F16) __syncthreads();
    for (int item = tid; item < 16 * ru * 4; item += kThreads) {
      const int row = item / (4 * ru), r8 = item % (4 * ru);
      f32x4 v[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
      if (row < t.rows && 2 * r8 < row4) {
        v[0] = s_sum[row * row4 + 2 * r8];
        v[1] = s_sum[row * row4 + 2 * r8 + 1];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)  // ranks behind the adapter's: not a number where x is not finite
        if (r8 * 8 + i >= rank) v[i / 4][i % 4] = 0.f;
      float inv = 1.f;
      if constexpr (F16) inv = 1.0f / s_scale[row];  // a power of two: exact
      u32x4 part[3];
      // The first part is the nearest number of the adapters' type: of sums from 2^128 - 2^119 on bf16's largest, as
      // the nearest is an infinity and the rest then no number.  What is not finite itself goes into the second part.
      constexpr float kMost = F16 ? 65504.0f : 0x1.fep127f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float rest = v[i / 4][i % 4] * inv;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const uint32_t b = lora_round<F16>(k == 0 ? __builtin_amdgcn_fmed3f(rest, -kMost, kMost) : rest);
          rest = k == 1 && !__builtin_isfinite(rest) ? 0.f : rest - lora_value<F16>(b);
          part[k][i / 2] = i % 2 ? part[k][i / 2] | b << 16 : b;
        }
      }
      uint8_t* o = s_t + (size_t)(r8 / 4) * kUpParts + ((r8 & 3) * 16 + row) * 16;
#pragma unroll
      for (int k = 0; k < 3; ++k) *(u32x4*)(o + 1024 * k) = part[k];
    }
  }
  __syncthreads();
  float* turn = (float*)s_work + wave * 16 * kTurnRow;
  for (int b = b0 + wave; b < b1; b += kWaves) {
    f32x4 acc[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int r = 0; r < ru; ++r) {
      u32x4 v[4];
#pragma unroll
      for (int f = 0; f < 4; ++f) v[f] = w[f];
      if (r + 1 < ru)
        load_w(b, r + 1);
      else if (b + kWaves < b1)
        load_w(b + kWaves, 0);
      const uint8_t* at = s_t + (size_t)r * kUpParts + lane * 16;
#pragma unroll
      for (int k = 2; k >= 0; --k) {  // the smallest parts first
        const u32x4 part = *(const u32x4*)(at + 1024 * k);
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[f] = lora_product<F16>(v[f], part, acc[f]);
      }
    }
    // acc: token lane % 16, features 16 f + 4 (lane / 16)..
    float m = 1.f;
    if constexpr (F16)
      if (ru) m = s_scale[lane & 15];
#pragma unroll
    for (int f = 0; f < 4; ++f) *(f32x4*)(turn + (lane & 15) * kTurnRow + 16 * f + 4 * (lane >> 4)) = acc[f] * m;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int n = b * 64 + n0;
    if constexpr (WHOLE) {
      float y[2][8];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float* from = turn + (half + 8 * i) * kTurnRow + n0;
        const f32x4 lo = *(const f32x4*)from, hi = *(const f32x4*)(from + 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          y[i][j] = j < 4 ? lo[j] : hi[j - 4];
        }
        if constexpr (BASE == 2) {
#pragma unroll
          for (int j = 0; j < 8; ++j) y[i][j] += __uint_as_float(base[2 * i + j / 4][j % 4]);
        } else if constexpr (BASE == 1) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            y[i][j] += __uint_as_float(j % 2 ? base[i][j / 2] & 0xffff0000u : base[i][j / 2] << 16);
        }
      }
      if (b + kWaves < b1) load_base(b + kWaves);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (half + 8 * i >= t.rows || n >= p.N) continue;
        const size_t at = (i ? at1 : at0) + n;
        if (p.out_f32) {
          *(f32x4*)((float*)p.out + at) = f32x4{y[i][0], y[i][1], y[i][2], y[i][3]};
          *(f32x4*)((float*)p.out + at + 4) = f32x4{y[i][4], y[i][5], y[i][6], y[i][7]};
        } else {
          u32x4 o;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            o[j] = mx_bf16x2(y[i][2 * j], y[i][2 * j + 1]);
          *(u32x4*)((uint16_t*)p.out + at) = o;
        }
      }
    } else {
      float y[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        y[i] = turn[i * kTurnRow + n0];
        if constexpr (BASE != 0) y[i] += __uint_as_float(base[i / 4][i % 4]);
      }
      if (b + kWaves < b1) load_base(b + kWaves);
      if (p.out_f32) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < t.rows && n < p.N) ((float*)p.out)[(size_t)order[i] * p.N + n] = y[i];
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < t.rows && n < p.N) ((uint16_t*)p.out)[(size_t)order[i] * p.N + n] = (uint16_t)mx_bf16x2(y[i], 0.f);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// ---------------------------------------------------------------- launches

static int up_div(int a, int b) { return (a + b - 1) / b; }

// Eight pieces, as far as each wave has two K-steps: one for each XCD, and few enough for the second launch, each
// of whose workgroups adds them up.
template <int TU>
static int pieces_of(int K) {
  return std::min(kLoraMaxPieces, up_div(K / 32, 2 * kDownWaves<TU, 1>));
}
// Half as many as long as the most tiles that a plan can hold are two workgroups a CU: 2048 tokens of 17408 and rank
// 64 with eight adapters, 73 tiles at most, take 22.8 us in four pieces, 25.0 in eight and 31.9 in 16 (and 31.8 in six,
// which no XCD has to itself).  That counts a tile for every adapter that is loaded, used or not, as the host knows no
// more: four requests there take 33 us (both launches) with 4 to 24 adapters loaded, 41 with 64 (two pieces) and 57-59
// with 200 to 1024 (one piece, 64 workgroups); 512 tokens 19, 23 and from 512 adapters on 55.
static int lora_pieces(int M, int K, int adapters, int num_cus) {
  int pieces = lora_tile(M) == 16 ? pieces_of<1>(K) : pieces_of<2>(K);
  while (pieces > 1 && pieces * lora_max_tiles(M, adapters) >= 2 * num_cus) pieces /= 2;
  return pieces;
}

static int padded_rank(int rank) { return (rank + 15) / 16 * 16; }

size_t lora_parts_bytes(int M, int K, int max_rank) {
  return align256((size_t)pieces_of<2>(K) * M * padded_rank(max_rank) * 4);  // the most of both kinds
}

template <bool F16, int TU, int RU>
static int launch_down(const LoraArgs& a, int max_tiles, int pieces, hipStream_t s) {
  constexpr size_t lds = kDownLds<TU, RU>;
  auto kern = lora_down_kernel<F16, TU, RU>;
  if constexpr (lds > 65536) {
    static std::atomic<uint64_t> raised{0};
    if (int rc = raise_lds_once((const void*)kern, (int)lds, raised)) return rc;
  }
  hipLaunchKernelGGL(kern, dim3(pieces, max_tiles), dim3(kDownWaves<TU, RU> * 64), lds, s, a, max_tiles,
                     padded_rank(a.max_rank));
  return check_launch("lora_down_kernel");
}

template <bool F16, bool WHOLE, int BASE, int DOWN>
static int launch_up(const LoraArgs& a, int max_tiles, int pieces, int num_cus, hipStream_t s) {
  const int blocks = up_div(a.N, 64), tile_units = lora_tile(a.M) / 16;
  const int tiles = std::max(1, std::min(max_tiles * tile_units / 2, up_div(a.M, 16)));
  // about a workgroup a CU, as far as each wave has a block: when the two launches took 44.1 us at 2048 tokens of
  // 17408 -> 5120 and rank 64 (39 now), two workgroups took 48.9 (each adds the pieces up again), one and two of four
  // waves 48.4 and 45.8
  const int slots = DOWN && max_tiles >= 8 ? up_div(max_tiles, 8) * 8 : max_tiles * tile_units;
  const int most = std::max(1, DOWN ? std::min(up_div(blocks, 4), num_cus / slots)
                                    : std::min(up_div(blocks, kUpWaves<0>), up_div(num_cus, tiles)));
  const int each = up_div(blocks, most), runs = up_div(blocks, each), units = padded_rank(a.max_rank) / 16;
  auto kern = lora_up_kernel<F16, WHOLE, BASE, DOWN>;
  if constexpr (lora_up_lds<DOWN>(kLoraMaxRank / 16) > 65536 - 64) {
    static std::atomic<uint64_t> raised{0};
    if (int rc = raise_lds_once((const void*)kern, (int)lora_up_lds<DOWN>(kLoraMaxRank / 16), raised)) return rc;
  }
  hipLaunchKernelGGL(kern, dim3(slots * runs), dim3(kUpWaves<DOWN> * 64), lora_up_lds<DOWN>(units), s, a,
                     max_tiles, units * 16, pieces, runs, each, tile_units);
  return check_launch("lora_up_kernel");
}
template <bool F16, bool WHOLE, int DOWN>
static int launch_up_base(const LoraArgs& a, int max_tiles, int pieces, int num_cus, hipStream_t s) {
  if (!a.base) return launch_up<F16, WHOLE, 0, DOWN>(a, max_tiles, pieces, num_cus, s);
  if (!a.base_f32) return launch_up<F16, WHOLE, 1, DOWN>(a, max_tiles, pieces, num_cus, s);
  return launch_up<F16, WHOLE, 2, DOWN>(a, max_tiles, pieces, num_cus, s);
}
template <bool F16, int DOWN>
static int launch_up_rows(const LoraArgs& a, int max_tiles, int pieces, int num_cus, hipStream_t s) {
  return a.N % 8 ? launch_up_base<F16, false, DOWN>(a, max_tiles, pieces, num_cus, s)
                 : launch_up_base<F16, true, DOWN>(a, max_tiles, pieces, num_cus, s);
}

// Whether t is made by every workgroup that uses it: where that reads at most half a megabyte of A and x, a third of
// that beyond 32 ranks.  One launch / two, us in a graph (and with the host's time in a loop of calls):
//   up to 32 ranks: one token of 5120 -> 5120 and rank 16, 174 KB: 6.8 / 7.5 (10.6 / 13.4); 5120 -> 17408 and rank 32,
//   492 KB: 16 tokens of 16 adapters 12.0 / 13.1 (11.7 / 13.5), of one 8.9 / 8.5 (10.4 / 13.4), of one of 16 loaded 12.1 /
//   8.7 (12.0 / 13.7), 32 tokens of twelve 11.6 / 11.0 (11.3 / 13.3): near the limit one launch is the host's gain;
//   one token of 17408 -> 5120 and rank 16, 592 KB: 10.9 / 7.9 (10.9 / 13.8);
//   rank 64: one token of 1024 -> 5120, 133 KB: 8.9 / 9.5 (10.4 / 13.6), 16 of 16 adapters, 164 KB: 11.9 / 11.2 (11.7 /
//   13.4); one token of 2048 -> 2048, 266 KB: 10.1 / 9.4 (10.7 / 13.8), of 5120 -> 5120, 666 KB: 14.7 / 9.6 (14.6 / 13.6);
//   rank 128 would bear a higher limit: one token of 1024 -> 5120, 264 KB: 9.3 / 11.4, 16 of 16 adapters 12.6 / 14.1; of
//   2048 -> 5120, 528 KB: 11.7 / 11.3.
static bool lora_one_launch(int M, int K, int max_rank) {
  const int ranks = padded_rank(max_rank);
  return lora_tile(M) == 16 && (size_t)(ranks + std::min(M, 16)) * K * 2 <= (ranks <= 32 ? 500000 : 167000);
}

LoraPath lora_path(int M, int K, int adapters, int max_rank, int num_cus) {
  const int units = padded_rank(max_rank) / 16, tile_units = lora_tile(M) / 16;
  return LoraPath{lora_one_launch(M, K, max_rank), tile_units, units <= 1 ? 1 : units <= 2 ? 2 : units <= 4 ? 4 : 8,
                  lora_pieces(M, K, adapters, num_cus), tile_units == 1 ? pieces_of<1>(K) : pieces_of<2>(K)};
}

template <bool F16, int TU>
static int launch_tokens(const LoraArgs& a, int num_cus, hipStream_t s) {
  const LoraPath path = lora_path(a.M, a.K, a.adapters, a.max_rank, num_cus);
  const int max_tiles = lora_max_tiles(a.M, a.adapters), pieces = path.pieces, units = path.rank_units;
  if (TU == 1 && path.one)
    return units == 1   ? launch_up_rows<F16, 1>(a, max_tiles, pieces, num_cus, s)
           : units == 2 ? launch_up_rows<F16, 2>(a, max_tiles, pieces, num_cus, s)
           : units == 4 ? launch_up_rows<F16, 4>(a, max_tiles, pieces, num_cus, s)
                        : launch_up_rows<F16, 8>(a, max_tiles, pieces, num_cus, s);
  const int rc = units == 1   ? launch_down<F16, TU, 1>(a, max_tiles, pieces, s)
                 : units == 2 ? launch_down<F16, TU, 2>(a, max_tiles, pieces, s)
                 : units == 4 ? launch_down<F16, TU, 4>(a, max_tiles, pieces, s)
                              : launch_down<F16, TU, 8>(a, max_tiles, pieces, s);
  if (rc) return rc;
  return launch_up_rows<F16, 0>(a, max_tiles, pieces, num_cus, s);
}

int launch_lora(const LoraArgs& a, int num_cus, hipStream_t s) {
  if (lora_tile(a.M) == 16) return a.f16 ? launch_tokens<true, 1>(a, num_cus, s) : launch_tokens<false, 1>(a, num_cus, s);
  return a.f16 ? launch_tokens<true, 2>(a, num_cus, s) : launch_tokens<false, 2>(a, num_cus, s);
}

}  // namespace qmlp
