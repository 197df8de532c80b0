// qmlp_lora_abi.hip -- the extern "C" entry points of the low-rank adapters (include/qwen_mlp.h): argument
// validation and dispatch.  No call allocates.
#include "../../include/qwen_mlp.h"
#include "qmlp_lora.h"

namespace qmlp {

static bool tokens_ok(int M) { return M >= 1 && M <= 65536; }
static bool adapters_ok(int n) { return n >= 1 && n <= kLoraMaxAdapters; }
static bool sizes_ok(int N, int K) { return N >= 1 && N <= kMaxDim && K >= 32 && K <= kMaxDim && K % 32 == 0; }
static bool rank_ok(int r) { return r >= 1 && r <= kLoraMaxRank; }
static bool overlap(const void* p, size_t n, const void* q, size_t m) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return p && q && a < b + m && b < a + n;
}

}  // namespace qmlp

using namespace qmlp;

extern "C" {

size_t qmlp_lora_plan_bytes(int M, int adapters) {
  return tokens_ok(M) && adapters_ok(adapters) ? lora_plan_words(M, adapters) * 4 : 0;
}

int qmlp_lora_plan(const int32_t* ids, int M, int adapters, void* plan, size_t plan_bytes, qmlp_stream_t stream) {
  const char* fn = "qmlp_lora_plan";
  if (!ids || !plan) return set_error(QMLP_E_NULL, "%s: null pointer", fn);
  if (!tokens_ok(M) || !adapters_ok(adapters))
    return set_error(QMLP_E_SHAPE, "%s: M=%d out of range [1, 65536] or %d adapters of [1, %d]", fn, M, adapters,
                     kLoraMaxAdapters);
  if ((uintptr_t)ids % 4 || !aligned16(plan)) return set_error(QMLP_E_ALIGN, "%s: misaligned pointer", fn);
  const size_t need = qmlp_lora_plan_bytes(M, adapters);
  if (plan_bytes < need)
    return set_error(QMLP_E_WORKSPACE, "%s: the plan holds %zu bytes, needs %zu", fn, plan_bytes, need);
  if (overlap(plan, need, ids, (size_t)M * 4)) return set_error(QMLP_E_SHAPE, "%s: the plan must not overlap ids", fn);
  DeviceInfo di;
  if (int rc = current_device_info(&di)) return rc;
  return launch_lora_plan(ids, M, adapters, (int*)plan, (hipStream_t)stream);
}

size_t qmlp_lora_workspace_bytes(int M, int K, int max_rank) {
  return tokens_ok(M) && sizes_ok(1, K) && rank_ok(max_rank) ? lora_parts_bytes(M, K, max_rank) : 0;
}

int qmlp_lora_path(int M, int N, int K, int adapters, int max_rank, int num_cus, int* out5) {
  const char* fn = "qmlp_lora_path";
  if (!out5) return set_error(QMLP_E_NULL, "%s: null pointer", fn);
  if (!tokens_ok(M) || !sizes_ok(N, K) || !adapters_ok(adapters) || !rank_ok(max_rank) || num_cus < 1)
    return set_error(QMLP_E_SHAPE, "%s: M=%d N=%d K=%d, %d adapters, rank %d on %d CUs", fn, M, N, K, adapters, max_rank,
                     num_cus);
  const LoraPath p = lora_path(M, K, adapters, max_rank, num_cus);
  out5[0] = p.one ? 1 : 2;
  out5[1] = p.tile_units;
  out5[2] = p.rank_units;
  out5[3] = p.one ? 1 : p.pieces;
  out5[4] = p.one ? 1 : p.most_pieces;
  return 0;
}

int qmlp_lora_linear(const void* x, int x_type, int64_t x_stride, const void* a, const void* b, const void* meta,
                     int adapters, int max_rank, const void* plan, const void* base, void* out, void* ws,
                     size_t ws_bytes, int M, int N, int K, int flags, qmlp_stream_t stream) {
  const char* fn = "qmlp_lora_linear";
  if (!x || !a || !b || !meta || !plan || !out || !ws) return set_error(QMLP_E_NULL, "%s: null pointer", fn);
  if (x_type != QMLP_X_BF16 && x_type != QMLP_X_F16)
    return set_error(QMLP_E_FORMAT, "%s: x must be bf16 or fp16 (type %d)", fn, x_type);
  if (flags & ~(QMLP_OUT_F32 | QMLP_RESIDUAL_F32)) return set_error(QMLP_E_FORMAT, "%s: bad flags 0x%x", fn, flags);
  if (!tokens_ok(M)) return set_error(QMLP_E_SHAPE, "%s: M=%d out of range [1, 65536]", fn, M);
  if (!sizes_ok(N, K))
    return set_error(QMLP_E_SHAPE, "%s: N=%d and K=%d must be positive, K a multiple of 32", fn, N, K);
  if (!adapters_ok(adapters) || !rank_ok(max_rank))
    return set_error(QMLP_E_SHAPE, "%s: %d adapters of [1, %d], rank %d of [1, %d]", fn, adapters, kLoraMaxAdapters,
                     max_rank, kLoraMaxRank);
  if (!aligned16(x) || !aligned16(a) || !aligned16(b) || !aligned16(meta) || !aligned16(plan) || !aligned16(base) ||
      !aligned16(out) || !aligned16(ws))
    return set_error(QMLP_E_ALIGN, "%s: every pointer must be 16-byte aligned", fn);
  if (x_stride < K || x_stride > (int64_t)1 << 40 || x_stride % 8)
    return set_error(QMLP_E_SHAPE, "%s: row stride %lld must be at least %d elements and a multiple of 16 bytes", fn,
                     (long long)x_stride, K);
  const size_t need = qmlp_lora_workspace_bytes(M, K, max_rank);
  if (ws_bytes < need)
    return set_error(QMLP_E_WORKSPACE, "%s: workspace holds %zu bytes, needs %zu", fn, ws_bytes, need);
  const bool out_f32 = (flags & QMLP_OUT_F32) != 0, base_f32 = (flags & QMLP_RESIDUAL_F32) != 0;
  const size_t ob = (size_t)M * N * (out_f32 ? 4 : 2), bb = (size_t)M * N * (base_f32 ? 4 : 2);
  const size_t xb = ((size_t)(M - 1) * (size_t)x_stride + K) * 2, pb = qmlp_lora_plan_bytes(M, adapters);
  if (base && base != out && overlap(out, ob, base, bb))
    return set_error(QMLP_E_SHAPE, "%s: out may equal base but must not partially overlap it", fn);
  if (base && base == out && out_f32 != base_f32)
    return set_error(QMLP_E_SHAPE, "%s: an in-place base needs the same dtype as out", fn);
  // a and b: their first bytes stand for them (their sizes follow from the ranks in meta)
  const void* ins[5] = {x, plan, meta, a, b};
  const size_t sizes[5] = {xb, pb, (size_t)adapters * 16, 16, 16};
  for (int i = 0; i < 5; ++i)
    if (overlap(out, ob, ins[i], sizes[i]) || overlap(ws, need, ins[i], sizes[i]))
      return set_error(QMLP_E_SHAPE, "%s: out and the workspace must not overlap an input", fn);
  if (overlap(ws, need, out, ob) || overlap(ws, need, base, bb))
    return set_error(QMLP_E_SHAPE, "%s: the workspace must not overlap another argument", fn);
  DeviceInfo di;
  if (int rc = current_device_info(&di)) return rc;
  const LoraArgs args{(const uint8_t*)x, (size_t)x_stride * 2, {(const uint8_t*)a, (const uint8_t*)b, (const int*)meta},
                      adapters, max_rank, (const int*)plan, base, out, (float*)ws, M, N, K,
                      x_type == QMLP_X_F16 ? 1 : 0, out_f32 ? 1 : 0, base_f32 ? 1 : 0};
  return launch_lora(args, di.num_cus, (hipStream_t)stream);
}

}  // extern "C"
