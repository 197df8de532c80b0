// qmlp_mx_abi.hip -- the extern "C" entry points of the MXFP4 operators, of their forms with 8-bit activations
// and of the norm in front of them (include/qwen_mlp.h), and the MXFP4 forward: argument validation,
// workspace layout, dispatch.  No call allocates.
#include <algorithm>

#include "../../include/qwen_mlp.h"
#include "qmlp_internal.h"
#include "qmlp_mx8.h"

namespace qmlp {

bool mx_shape_ok(int rows, int cols) {
  return rows > 0 && cols > 0 && cols % kMxBlock == 0 && rows <= kMaxDim && cols <= kMaxDim;
}

static bool mx_tokens_ok(int M) { return M >= 1 && M <= 65536; }

// Forward workspace: the arrival counters that every format's workspace starts with (a pool's
// workspace may serve other formats in turn; these kernels leave them alone), the quantised x and h, and
// for many tokens the partial tiles of split K ranges, which both products use in turn.
static size_t part_bytes(int M) { return M > kMxFewTokens ? kMxPartBytes : 0; }
// The type of packed activations, and their bytes.
static int packed_type(bool a8) { return a8 ? QMLP_X_MXINT8 : QMLP_X_MXFP4; }
static size_t units_bytes(int rows, int cols, bool a8) {
  return a8 ? mx8_units_bytes(rows, cols) : mx_units_bytes(rows, cols);
}
// Unpacked rows that the product does not quantise by itself.
static size_t packed_x_bytes(int M, int K, int x_type, bool a8) {
  return x_type == packed_type(a8) || mx_quantizes_inside(M, K, a8) ? 0 : align256(units_bytes(M, K, a8));
}
struct MxWs {
  size_t x, h, parts, total;
};
static MxWs mx_ws(int M, int H, int I) {
  MxWs L{};
  L.x = align256(QMLP_WS_COUNTER_BYTES);
  L.h = L.x + align256(mx_units_bytes(M, H));
  L.parts = L.h + align256(mx_units_bytes(M, I));
  L.total = L.parts + part_bytes(M);
  return L;
}
size_t mx_forward_bytes(int M, int H, int I) { return mx_ws(M, H, I).total; }

// One product as planned for its sizes; unpacked rows are quantised into packed_x first unless the
// kernel does that itself.
static int run_product(MxProduct p, void* packed_x, int num_cus, hipStream_t s) {
  const MxPlan plan = mx_plan(p.o.M, p.o.N, p.K, p.mode == kMxRowsOut ? 1 : 2, num_cus, p.a8);
  const int packed = packed_type(p.a8);
  if (p.x_type != packed && !mx_quantizes_inside(p.o.M, p.K, p.a8)) {
    if (int rc = p.a8 ? launch_mx8_quantize(p.x, p.x_type, p.row_bytes, p.o.M, p.K, packed_x, s)
                      : launch_mx_quantize(p.x, p.x_type, p.row_bytes, p.o.M, p.K, packed_x, s))
      return rc;
    p.x = (const uint8_t*)packed_x;
    p.x_type = packed;
  }
  if (p.x_type == packed) p.x_type = kMxPackedX;  // the kernels know one packed type, that of their format
  if (plan.kind == kMxFew) return launch_mx8_few(p, plan, s);
  return plan.kind == kMxTiles ? launch_mx_tiled(p, plan, s) : launch_mx_stream(p, plan, s);
}

int mx_forward(const void* x, const void* wg, const void* wu, const void* wd, const void* residual, void* out, void* ws,
               int M, int H, int I, int flags, const void* normw, float eps, int num_cus, hipStream_t s) {
  const MxWs L = mx_ws(M, H, I);
  uint8_t* base = (uint8_t*)ws;
  MxProduct gu{(const uint8_t*)x, (const uint8_t*)wg, (const uint8_t*)wu, H, kMxPacked,
               {base + L.h, nullptr, M, I, 0, 0}, 0, QMLP_X_BF16, (size_t)H * 2, base + L.parts};
  if (normw) {
    if (int rc = launch_mx_norm_quantize(x, (size_t)H * 2, normw, eps, M, H, base + L.x, s)) return rc;
    gu.x = base + L.x;
    gu.x_type = QMLP_X_MXFP4;
  }
  if (int rc = run_product(gu, base + L.x, num_cus, s)) return rc;
  MxProduct down{base + L.h, (const uint8_t*)wd, nullptr, I, kMxRowsOut,
                 {out, residual, M, H, (flags & QMLP_OUT_F32) ? 1 : 0, (flags & QMLP_RESIDUAL_F32) ? 1 : 0},
                 1, QMLP_X_MXFP4, 0, base + L.parts};
  return run_product(down, nullptr, num_cus, s);
}

// [p, p + n) and [q, q + m) have a byte in common.
static bool overlap(const void* p, size_t n, const void* q, size_t m) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return p && q && a < b + m && b < a + n;
}

static size_t x_size(int type) { return type == QMLP_X_F32 ? 4 : 2; }

// Checks an unpacked activation matrix.
static int check_rows(const char* fn, const void* x, int type, int64_t stride, int K) {
  if (type != QMLP_X_BF16 && type != QMLP_X_F16 && type != QMLP_X_F32)
    return set_error(QMLP_E_FORMAT, "%s: unknown activation type %d", fn, type);
  if (!aligned16(x)) return set_error(QMLP_E_ALIGN, "%s: x must be 16-byte aligned", fn);
  if (stride < K || stride > (int64_t)1 << 40 || stride * (int64_t)x_size(type) % 16)
    return set_error(QMLP_E_SHAPE, "%s: row stride %lld must be at least %d elements and a multiple of 16 bytes", fn,
                     (long long)stride, K);
  return 0;
}
static size_t rows_extent(int type, int64_t stride, int M, int K) {
  return ((size_t)(M - 1) * (size_t)stride + K) * x_size(type);
}

// The products: a8 selects 8-bit activations; gate_add and up_add belong to their gate/up pair.
static int product_impl(const char* fn, bool a8, const void* x, int x_type, int64_t x_stride, const void* w0,
                        const void* w1, int nmat, const void* residual, const void* gate_add, const void* up_add,
                        void* out, void* ws, size_t ws_bytes, int M, int N, int K, int flags, hipStream_t s) {
  if (!x || !w0 || (nmat > 1 && !w1) || !out) return set_error(QMLP_E_NULL, "%s: null pointer", fn);
  const int out_packed = a8 ? QMLP_OUT_MXINT8 : QMLP_OUT_MXFP4, x_packed = packed_type(a8);
  const int known = nmat > 1 ? (QMLP_OUT_F32 | out_packed) : (QMLP_OUT_F32 | QMLP_RESIDUAL_F32);
  if ((flags & ~known) || ((flags & QMLP_OUT_F32) && (flags & out_packed)))
    return set_error(QMLP_E_FORMAT, "%s: bad flags 0x%x", fn, flags);
  if (!mx_tokens_ok(M)) return set_error(QMLP_E_SHAPE, "%s: M=%d out of range [1, 65536]", fn, M);
  if (!mx_shape_ok(N, K))
    return set_error(QMLP_E_SHAPE, "%s: N=%d and K=%d must be positive, K a multiple of 32", fn, N, K);
  const bool packed_out = (flags & out_packed) != 0;
  if (packed_out && N % kMxK)
    return set_error(QMLP_E_SHAPE, "%s: a packed output needs N=%d to be a multiple of 256", fn, N);
  if (!aligned16(x) || !aligned16(w0) || !aligned16(w1) || !aligned16(residual) || !aligned16(out) || !aligned16(ws) ||
      !aligned16(gate_add) || !aligned16(up_add))
    return set_error(QMLP_E_ALIGN, "%s: every pointer must be 16-byte aligned", fn);
  if (x_type != x_packed)
    if (int rc = check_rows(fn, x, x_type, x_stride, K)) return rc;
  const size_t xbytes = x_type == x_packed ? units_bytes(M, K, a8) : rows_extent(x_type, x_stride, M, K);
  const size_t obytes = packed_out ? units_bytes(M, N, a8) : (size_t)M * N * ((flags & QMLP_OUT_F32) ? 4 : 2);
  const size_t wbytes = mx_units_bytes(N, K), rbytes = (size_t)M * N * ((flags & QMLP_RESIDUAL_F32) ? 4 : 2);
  if (overlap(out, obytes, x, xbytes) || overlap(out, obytes, w0, wbytes) || overlap(out, obytes, w1, wbytes))
    return set_error(QMLP_E_SHAPE, "%s: out must not overlap x or a weight", fn);
  if (residual && residual != out && overlap(out, obytes, residual, rbytes))
    return set_error(QMLP_E_SHAPE, "%s: out may equal residual but must not partially overlap it", fn);
  if (residual && residual == out && ((flags & QMLP_OUT_F32) != 0) != ((flags & QMLP_RESIDUAL_F32) != 0))
    return set_error(QMLP_E_SHAPE, "%s: an in-place residual needs the same dtype as out", fn);
  const size_t abytes = (size_t)M * N * 4;
  if (overlap(out, obytes, gate_add, abytes) || overlap(out, obytes, up_add, abytes))
    return set_error(QMLP_E_SHAPE, "%s: out must not overlap gate_add or up_add", fn);
  const size_t need = a8 ? qmlp_w4a8_workspace_bytes(M, N, K, x_type) : qmlp_mx_workspace_bytes(M, N, K, x_type);
  if (need && !ws) return set_error(QMLP_E_NULL, "%s: null workspace", fn);
  if (ws_bytes < need)
    return set_error(QMLP_E_WORKSPACE, "%s: workspace holds %zu bytes, needs %zu", fn, ws_bytes, need);
  if (overlap(ws, need, x, xbytes) || overlap(ws, need, out, obytes) || overlap(ws, need, residual, rbytes) ||
      overlap(ws, need, w0, wbytes) || overlap(ws, need, w1, wbytes) || overlap(ws, need, gate_add, abytes) ||
      overlap(ws, need, up_add, abytes))
    return set_error(QMLP_E_SHAPE, "%s: the workspace must not overlap another argument", fn);
  DeviceInfo di;
  if (int rc = current_device_info(&di)) return rc;
  MxProduct p{(const uint8_t*)x, (const uint8_t*)w0, (const uint8_t*)w1, K,
              nmat == 1 ? kMxRowsOut : !packed_out ? kMxGated : a8 ? kMxPacked8 : kMxPacked,
              {out, residual, M, N, (flags & QMLP_OUT_F32) ? 1 : 0, (flags & QMLP_RESIDUAL_F32) ? 1 : 0,
               (const float*)gate_add, (const float*)up_add},
              -1, x_type, (size_t)x_stride * x_size(x_type), (uint8_t*)ws + packed_x_bytes(M, K, x_type, a8), a8};
  return run_product(p, ws, di.num_cus, s);
}

}  // namespace qmlp

using namespace qmlp;

extern "C" {

size_t qmlp_mx_workspace_bytes(int M, int N, int K, int x_type) {
  if (!mx_tokens_ok(M) || !mx_shape_ok(N, K)) return 0;
  return packed_x_bytes(M, K, x_type, false) + part_bytes(M);
}

size_t qmlp_w4a8_workspace_bytes(int M, int N, int K, int x_type) {
  if (!mx_tokens_ok(M) || !mx_shape_ok(N, K)) return 0;
  return packed_x_bytes(M, K, x_type, true) + part_bytes(M);
}

static int plan_impl(const char* fn, bool a8, int M, int N, int K, int nmat, int num_cus, int* out5) {
  if (!out5) return set_error(QMLP_E_NULL, "%s: null pointer", fn);
  if (!mx_tokens_ok(M) || !mx_shape_ok(N, K) || nmat < 1 || nmat > 2 || num_cus < 1)
    return set_error(QMLP_E_SHAPE, "%s: M=%d N=%d K=%d, %d matrices on %d CUs", fn, M, N, K, nmat, num_cus);
  const MxPlan p = mx_plan(M, N, K, nmat, num_cus, a8);
  out5[0] = p.kind == kMxTiles ? kMxStreamWide + p.height : p.kind == kMxFew ? 8 : (int)p.kind;
  out5[1] = p.ks;
  out5[2] = p.workgroups;
  out5[3] = (int)(p.part_bytes >> 10);
  out5[4] = mx_quantizes_inside(M, K, a8) ? 1 : 0;
  return 0;
}

int qmlp_mx_plan(int M, int N, int K, int nmat, int num_cus, int* out5) {
  return plan_impl("qmlp_mx_plan", false, M, N, K, nmat, num_cus, out5);
}

int qmlp_w4a8_plan(int M, int N, int K, int nmat, int num_cus, int* out5) {
  return plan_impl("qmlp_w4a8_plan", true, M, N, K, nmat, num_cus, out5);
}

static int quantize_checks(const char* fn, bool a8, const void* x, int x_type, int64_t x_stride, int rows, int cols,
                           const void* packed, size_t packed_bytes) {
  if (!x || !packed) return set_error(QMLP_E_NULL, "%s: null pointer", fn);
  if (!mx_shape_ok(rows, cols))
    return set_error(QMLP_E_SHAPE, "%s: cols must be a multiple of 32 (%dx%d)", fn, rows, cols);
  if (int rc = check_rows(fn, x, x_type, x_stride, cols)) return rc;
  if (!aligned16(packed)) return set_error(QMLP_E_ALIGN, "%s: misaligned pointer", fn);
  const size_t need = units_bytes(rows, cols, a8);
  if (packed_bytes < need)
    return set_error(QMLP_E_WORKSPACE, "%s: packed buffer holds %zu bytes, needs %zu", fn, packed_bytes, need);
  if (overlap(packed, need, x, rows_extent(x_type, x_stride, rows, cols)))
    return set_error(QMLP_E_SHAPE, "%s: the packed buffer must not overlap x", fn);
  return 0;
}

int qmlp_mx_quantize(const void* x, int x_type, int64_t x_stride, int rows, int cols, void* packed,
                     size_t packed_bytes, qmlp_stream_t stream) {
  if (int rc = quantize_checks("qmlp_mx_quantize", false, x, x_type, x_stride, rows, cols, packed, packed_bytes)) return rc;
  DeviceInfo di;
  if (int rc = current_device_info(&di)) return rc;
  return launch_mx_quantize(x, x_type, (size_t)x_stride * x_size(x_type), rows, cols, packed, (hipStream_t)stream);
}

int qmlp_mx_quantize_rmsnorm(const void* h, int64_t h_stride, const void* norm_w, float eps, int rows, int cols,
                             void* packed, size_t packed_bytes, qmlp_stream_t stream) {
  const char* fn = "qmlp_mx_quantize_rmsnorm";
  if (!norm_w) return set_error(QMLP_E_NULL, "%s: null norm weight", fn);
  if (!aligned16(norm_w)) return set_error(QMLP_E_ALIGN, "%s: misaligned norm weight", fn);
  if (!(eps >= 0.0f)) return set_error(QMLP_E_SHAPE, "%s: eps must be >= 0", fn);
  if (int rc = quantize_checks(fn, false, h, QMLP_X_BF16, h_stride, rows, cols, packed, packed_bytes)) return rc;
  if (overlap(packed, mx_units_bytes(rows, cols), norm_w, (size_t)cols * 2))
    return set_error(QMLP_E_SHAPE, "%s: the packed buffer must not overlap the norm weight", fn);
  DeviceInfo di;
  if (int rc = current_device_info(&di)) return rc;
  return launch_mx_norm_quantize(h, (size_t)h_stride * 2, norm_w, eps, rows, cols, packed, (hipStream_t)stream);
}

static int dequantize_impl(const char* fn, bool a8, const void* packed, int rows, int cols, void* out, int out_type,
                           hipStream_t s) {
  if (!packed || !out) return set_error(QMLP_E_NULL, "%s: null pointer", fn);
  if (out_type != QMLP_X_BF16 && out_type != QMLP_X_F32)
    return set_error(QMLP_E_FORMAT, "%s: unknown output type %d", fn, out_type);
  if (!mx_shape_ok(rows, cols))
    return set_error(QMLP_E_SHAPE, "%s: cols must be a multiple of 32 (%dx%d)", fn, rows, cols);
  if (!aligned16(packed) || !aligned16(out)) return set_error(QMLP_E_ALIGN, "%s: misaligned pointer", fn);
  if (overlap(packed, units_bytes(rows, cols, a8), out, (size_t)rows * cols * x_size(out_type)))
    return set_error(QMLP_E_SHAPE, "%s: out must not overlap the packed buffer", fn);
  DeviceInfo di;
  if (int rc = current_device_info(&di)) return rc;
  return a8 ? launch_mx8_dequantize(packed, rows, cols, out, out_type == QMLP_X_F32, s)
            : launch_mx_dequantize(packed, rows, cols, out, out_type == QMLP_X_F32, s);
}

int qmlp_mx_dequantize(const void* packed, int rows, int cols, void* out, int out_type, qmlp_stream_t stream) {
  return dequantize_impl("qmlp_mx_dequantize", false, packed, rows, cols, out, out_type, (hipStream_t)stream);
}

size_t qmlp_mxint8_bytes(int rows, int cols) { return mx_shape_ok(rows, cols) ? mx8_units_bytes(rows, cols) : 0; }

int qmlp_mxint8_quantize(const void* x, int x_type, int64_t x_stride, int rows, int cols, void* packed,
                         size_t packed_bytes, qmlp_stream_t stream) {
  if (int rc = quantize_checks("qmlp_mxint8_quantize", true, x, x_type, x_stride, rows, cols, packed, packed_bytes))
    return rc;
  DeviceInfo di;
  if (int rc = current_device_info(&di)) return rc;
  return launch_mx8_quantize(x, x_type, (size_t)x_stride * x_size(x_type), rows, cols, packed, (hipStream_t)stream);
}

int qmlp_mxint8_dequantize(const void* packed, int rows, int cols, void* out, int out_type, qmlp_stream_t stream) {
  return dequantize_impl("qmlp_mxint8_dequantize", true, packed, rows, cols, out, out_type, (hipStream_t)stream);
}

int qmlp_mxint8_unpack(const void* packed, int rows, int cols, void* q, void* scales, qmlp_stream_t stream) {
  const char* fn = "qmlp_mxint8_unpack";
  if (!packed || !q || !scales) return set_error(QMLP_E_NULL, "%s: null pointer", fn);
  if (!mx_shape_ok(rows, cols))
    return set_error(QMLP_E_SHAPE, "%s: cols must be a multiple of 32 (%dx%d)", fn, rows, cols);
  if (!aligned16(packed) || !aligned16(q)) return set_error(QMLP_E_ALIGN, "%s: misaligned pointer", fn);
  const size_t need = mx8_units_bytes(rows, cols), qn = (size_t)rows * cols, sn = qn / kMxBlock;
  if (overlap(packed, need, q, qn) || overlap(packed, need, scales, sn) || overlap(q, qn, scales, sn))
    return set_error(QMLP_E_SHAPE, "%s: the buffers must not overlap", fn);
  DeviceInfo di;
  if (int rc = current_device_info(&di)) return rc;
  return launch_mx8_unpack(packed, rows, cols, q, scales, (hipStream_t)stream);
}

int qmlp_add_rmsnorm(const void* x, int x_type, int64_t x_stride, const void* residual, int residual_type,
                     int64_t residual_stride, const void* norm_w, float eps, int rows, int cols, void* h,
                     int64_t h_stride, void* n, void* packed, size_t packed_bytes, qmlp_stream_t stream) {
  const char* fn = "qmlp_add_rmsnorm";
  if (!x || !norm_w || (residual && !h) || (!n && !packed)) return set_error(QMLP_E_NULL, "%s: null pointer", fn);
  if (!mx_shape_ok(rows, cols))
    return set_error(QMLP_E_SHAPE, "%s: cols must be a multiple of 32 (%dx%d)", fn, rows, cols);
  if (x_type == QMLP_X_F16 || (residual && residual_type != QMLP_X_BF16 && residual_type != QMLP_X_F32))
    return set_error(QMLP_E_FORMAT, "%s: x and residual must be bf16 or fp32", fn);
  if (!(eps >= 0.0f)) return set_error(QMLP_E_SHAPE, "%s: eps must be >= 0", fn);
  if (int rc = check_rows(fn, x, x_type, x_stride, cols)) return rc;
  if (residual) {
    if (int rc = check_rows(fn, residual, residual_type, residual_stride, cols)) return rc;
    if (int rc = check_rows(fn, h, residual_type, h_stride, cols)) return rc;
  } else if (h) {
    return set_error(QMLP_E_NULL, "%s: h is the sum with a residual: null without one", fn);
  }
  if (!aligned16(norm_w) || !aligned16(n) || !aligned16(packed))
    return set_error(QMLP_E_ALIGN, "%s: every pointer must be 16-byte aligned", fn);
  const size_t need = mx8_units_bytes(rows, cols);
  if (packed && packed_bytes < need)
    return set_error(QMLP_E_WORKSPACE, "%s: packed buffer holds %zu bytes, needs %zu", fn, packed_bytes, need);
  const size_t xb = rows_extent(x_type, x_stride, rows, cols), wb = (size_t)cols * 2, nb = (size_t)rows * cols * 2;
  const size_t rb = residual ? rows_extent(residual_type, residual_stride, rows, cols) : 0;
  const size_t hb = residual ? rows_extent(residual_type, h_stride, rows, cols) : 0;
  if (h != residual || h_stride != residual_stride)
    if (overlap(h, hb, residual, rb))
      return set_error(QMLP_E_SHAPE, "%s: h may be the residual itself but must not overlap it otherwise", fn);
  const void* outs[3] = {h, n, packed};
  const size_t sizes[3] = {hb, nb, need};
  for (int i = 0; i < 3; ++i) {
    if (overlap(outs[i], sizes[i], x, xb) || overlap(outs[i], sizes[i], norm_w, wb) ||
        (i > 0 && overlap(outs[i], sizes[i], residual, rb)))
      return set_error(QMLP_E_SHAPE, "%s: an output must not overlap an input", fn);
    for (int j = 0; j < i; ++j)
      if (overlap(outs[i], sizes[i], outs[j], sizes[j]))
        return set_error(QMLP_E_SHAPE, "%s: the outputs must not overlap", fn);
  }
  DeviceInfo di;
  if (int rc = current_device_info(&di)) return rc;
  const AddNorm a{(const uint8_t*)x, (const uint8_t*)residual, (const uint16_t*)norm_w, (uint8_t*)h, (uint16_t*)n,
                  (uint8_t*)packed, (size_t)x_stride * x_size(x_type),
                  residual ? (size_t)residual_stride * x_size(residual_type) : 0,
                  residual ? (size_t)h_stride * x_size(residual_type) : 0, eps, rows, cols, x_type, residual_type};
  return launch_add_norm(a, (hipStream_t)stream);
}

int qmlp_mx_linear(const void* x, int x_type, int64_t x_stride, const void* w, const void* residual, void* out,
                   void* ws, size_t ws_bytes, int M, int N, int K, int flags, qmlp_stream_t stream) {
  return product_impl("qmlp_mx_linear", false, x, x_type, x_stride, w, nullptr, 1, residual, nullptr, nullptr, out, ws, ws_bytes, M, N, K,
                      flags, (hipStream_t)stream);
}

int qmlp_mx_swiglu(const void* x, int x_type, int64_t x_stride, const void* wg, const void* wu, void* out, void* ws,
                   size_t ws_bytes, int M, int N, int K, int flags, qmlp_stream_t stream) {
  return product_impl("qmlp_mx_swiglu", false, x, x_type, x_stride, wg, wu, 2, nullptr, nullptr, nullptr, out, ws, ws_bytes, M, N, K, flags,
                      (hipStream_t)stream);
}

int qmlp_w4a8_linear(const void* x, int x_type, int64_t x_stride, const void* w, const void* residual, void* out,
                     void* ws, size_t ws_bytes, int M, int N, int K, int flags, qmlp_stream_t stream) {
  return product_impl("qmlp_w4a8_linear", true, x, x_type, x_stride, w, nullptr, 1, residual, nullptr, nullptr, out, ws,
                      ws_bytes, M, N, K, flags, (hipStream_t)stream);
}

int qmlp_w4a8_swiglu(const void* x, int x_type, int64_t x_stride, const void* wg, const void* wu, const float* gate_add,
                     const float* up_add, void* out, void* ws, size_t ws_bytes, int M, int N, int K, int flags,
                     qmlp_stream_t stream) {
  return product_impl("qmlp_w4a8_swiglu", true, x, x_type, x_stride, wg, wu, 2, nullptr, gate_add, up_add, out, ws,
                      ws_bytes, M, N, K, flags, (hipStream_t)stream);
}

}  // extern "C"
