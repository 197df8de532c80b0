// qmlp_lora.h -- low-rank adapters of many requests at once: layouts and declarations.
//
//   out[m] = base[m] + s_a B_a (A_a x[m]),   a = ids[m];  A_a [r, K], B_a [N, r], s_a a number
//
// An adapter's matrices are used in the order of the 16x16x32 product's operands:
//   A: units of 16 ranks x 32 K, [rank unit][K / 32][lane][8]: lane l holds rank l % 16, K 8 (l / 16)..;
//   B: blocks of 64 features, [block][32 ranks][4][lane][8]: in part f lane l holds ranks 8 (l / 16).. of feature
//      16 f + l % 16 (features behind N and ranks behind the adapter's: zeros, the latter never read).
// Adapters follow each other.  The meta table holds {rank, rank units before in A, s_a's bits, 32s of ranks
// before in B} of each.
//
// A plan groups a batch's tokens by adapter: {magic, M, adapters, tiles}, then one {adapter, first row, rows, 0}
// per tile (rows: places in the order below, at most lora_tile(M) of one adapter; -1: without), then the tokens
// in that order.
#pragma once
#include "qmlp_internal.h"

namespace qmlp {

constexpr int kLoraMaxRank = 128;
constexpr int kLoraMaxAdapters = 1024;
constexpr int kLoraMagic = 0x41524f4c;
constexpr int kLoraMaxPieces = 8;

// Tokens of a tile.  One unit of 16 for few tokens (as a rule of as many requests); two share what they read
// of the adapters for many.
__host__ __device__ inline int lora_tile(int M) { return M <= 64 ? 16 : 32; }
inline int lora_max_tiles(int M, int adapters) {
  const int groups = M < adapters + 1 ? M : adapters + 1;
  return M / lora_tile(M) + groups;
}
inline size_t lora_plan_words(int M, int adapters) { return 4 + 4 * (size_t)lora_max_tiles(M, adapters) + M; }

struct LoraStack {
  const uint8_t* a;
  const uint8_t* b;
  const int* meta;
};
struct LoraArgs {
  const uint8_t* x;
  size_t x_bytes;  // from row to row
  LoraStack stack;
  int adapters, max_rank;
  const int* plan;
  const void* base;  // may be null
  void* out;
  float* parts;  // [piece][place][ranks padded to 16] sums over the pieces' K ranges
  int M, N, K;
  int f16, out_f32, base_f32;
};

// How a call runs for its sizes: whether in one launch, units of 16 tokens of a tile, the most units of 16 ranks that the
// kernels are made for, and (two launches) the pieces of the K range, a workgroup each, of the most that K would give.
struct LoraPath {
  bool one;
  int tile_units, rank_units, pieces, most_pieces;
};
LoraPath lora_path(int M, int K, int adapters, int max_rank, int num_cus);
size_t lora_parts_bytes(int M, int K, int max_rank);
int launch_lora_plan(const int* ids, int M, int adapters, int* plan, hipStream_t s);
int launch_lora(const LoraArgs& a, int num_cus, hipStream_t s);

}  // namespace qmlp
