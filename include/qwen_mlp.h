/*
 * qwen_mlp.h -- C ABI of libqwen_mlp.so, the MI355X (gfx950) fused Qwen3 SwiGLU MLP.
 *
 *   out = residual + down( silu(gate(x)) * up(x) )          (residual optional)
 *
 * Every pointer is a device pointer unless stated otherwise; every buffer is owned by the caller;
 * the library never allocates or frees device memory.  Work is enqueued on the given HIP stream
 * (nullptr = the legacy default stream), nothing synchronises the host unless stated, and no
 * call allocates, so the forward entry points can be captured in a HIP graph.
 *
 * Return codes: QMLP_OK (0) or a negative QMLP_E_* code; qmlp_last_error() then returns a
 * thread-local message naming the failing argument.
 *
 * Weight formats:
 *   QMLP_FMT_BF16  bf16 weights, bf16 matrix-core products, fp32 accumulation.
 *   QMLP_FMT_BFP8  bfp8 block float: 16 consecutive K values share one 8-bit exponent, each value
 *                  1 sign + 7 magnitude bits; dequantised in registers to fp16 matrix-core
 *                  operands, fp32 accumulation.
 *   QMLP_FMT_BF4   bf4 block float: the same 16-value groups with 1 sign + 3 magnitude bits
 *                  (0.5625 B/value).  In qmlp_forward it names the reference's mixed layout
 *                  (mlp.py:17-19,164-169): gate_proj and up_proj packed bf4, down_proj packed bfp8.
 *   QMLP_FMT_MXFP4 microscaled 4-bit floating point (OCP MX): 32 consecutive K values share one
 *                  power-of-two scale byte, each value is one of 0, .5, 1, 1.5, 2, 3, 4, 6 with a
 *                  sign (0.53125 B/value).  The activations are quantised to the same format in
 *                  every call, so both operands go to the scaled matrix-core products as they are
 *                  (fp32 accumulation); h, between the projections, is quantised once from fp32.
 * Weights are used in the library's packed ("tiled") layout, produced once by qmlp_pack().
 * Matrices are row-major [out_features, in_features] like the HF checkpoint tensors
 * gate_proj.weight [I,H], up_proj.weight [I,H], down_proj.weight [H,I].
 */
#ifndef QWEN_MLP_H
#define QWEN_MLP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* qmlp_stream_t; /* == hipStream_t */

#define QMLP_OK 0
#define QMLP_E_SHAPE (-1)     /* bad dimension (H, I, M, rows, cols) */
#define QMLP_E_ALIGN (-2)     /* pointer not 16-byte aligned */
#define QMLP_E_FORMAT (-3)    /* unknown format, or packed data that does not fit the format */
#define QMLP_E_LAUNCH (-4)    /* HIP launch / runtime error */
#define QMLP_E_WORKSPACE (-5) /* workspace too small */
#define QMLP_E_NULL (-6)      /* required pointer is null */
#define QMLP_E_DEVICE (-7)    /* no usable gfx950 device */

#define QMLP_FMT_BF16 0
#define QMLP_FMT_BFP8 1
#define QMLP_FMT_BF4 2
#define QMLP_FMT_MXFP4 4

/* Message for the last failing call on this host thread ("" if none).  Host only. */
const char* qmlp_last_error(void);

/* Library version string, "qwen_mlp <version> gfx950 src=<digest>": the digest (16 hex digits) is
 * the sha256 of the kernel sources and this header that the build compiled.  Host only. */
const char* qmlp_version(void);

/* ---------------------------------------------------------------- weight preparation (load time)
 *
 * The reference converts host bf16 tensors into device block-float tiles once per model
 * (docker/qwen-c2-graft/graft/mlp.py:125-169, ttnn.as_tensor(..., dtype=bfloat8_b/bfloat4_b,
 * layout=TILE_LAYOUT)); these calls are that step.
 */

/* Canonical bfp8 quantisation of a bf16 matrix w[rows, cols] (row-major, K = cols).
 * q: int8 [rows, cols]; e8: uint8 [rows, cols/16] (scale 2^(e8-127), 0 = zero group).
 * bad_groups (device uint32, nullable): incremented once per group holding a non-finite value.
 * Replaces the host quantiser inside ttnn.as_tensor(dtype=bfloat8_b) (mlp.py:155-162). */
int qmlp_quantize_bfp8(const void* w_bf16, int rows, int cols, void* q, void* e8,
                       uint32_t* bad_groups, qmlp_stream_t stream);

/* Canonical bf4 quantisation: as qmlp_quantize_bfp8 with magnitudes in [0, 7] (q in [-7, 7],
 * scale 2^(e8-127) with e8 = exponent of the group maximum + 127 - 3).  Replaces the host
 * quantiser inside ttnn.as_tensor(dtype=bfloat4_b) (mlp.py:17-19,164-169). */
int qmlp_quantize_bf4(const void* w_bf16, int rows, int cols, void* q, void* e8,
                      uint32_t* bad_groups, qmlp_stream_t stream);

/* Bytes of the packed device buffer for one [rows, cols] matrix (host only, no GPU needed): rows a
 * multiple of 16 and cols of 256; QMLP_FMT_MXFP4: any rows, cols a multiple of 32. */
size_t qmlp_packed_bytes(int rows, int cols, int fmt);

/* Pack one matrix into the library's tiled layout.
 *   fmt == QMLP_FMT_BFP8 or QMLP_FMT_BF4: src0 = q (int8 [rows,cols]), src1 = e8 (uint8
 *   [rows,cols/16]) from the matching quantiser.
 *   fmt == QMLP_FMT_BF16: src0 = bf16 [rows,cols], src1 unused (may be null).
 *   fmt == QMLP_FMT_MXFP4: src0 = codes (uint8 [rows,cols/2], the even K in the low half of a byte),
 *   src1 = scales (uint8 [rows,cols/32], 2^(s-127)), as microscaled checkpoints hold them; the
 *   trailer counts the scales of 255 (not a number) as groups with non-finite values.
 * packed must hold qmlp_packed_bytes(rows, cols, fmt) bytes.  The trailer of the packed buffer
 * records the largest row L2 norm and the number of bfp8 groups too small to keep (see
 * qmlp_packed_info); a nonzero count means the packed matrix is not lossless.
 * Replaces _build_gate_up / load_mlp_weights' tile conversion (mlp.py:23-42, 125-169). */
int qmlp_pack(const void* src0, const void* src1, int rows, int cols, int fmt, void* packed,
              size_t packed_bytes, qmlp_stream_t stream);

/* Reads the packed trailer back to host memory: largest row L2 norm (of the dequantised rows)
 * and count of flushed bfp8 groups (QMLP_FMT_MXFP4: both 0, its kernels need no bound and keep every
 * group).  Synchronises `stream`.  Load-time only. */
int qmlp_packed_info(const void* packed, int rows, int cols, int fmt, double* max_row_norm,
                     uint32_t* flushed_groups, qmlp_stream_t stream);

/* qmlp_quantize_bfp8 / _bf4 and qmlp_pack in one pass: bf16 [rows,cols] -> the same packed bytes in
 * any format, without the canonical intermediates.  qmlp_quantize_pack_info reads the trailer back
 * like qmlp_packed_info and also the number of groups that hold a non-finite value (packed as
 * zeros, with QMLP_FMT_MXFP4 as NaN; a matrix with such groups must not be used; always 0 for
 * QMLP_FMT_BF16). */
int qmlp_quantize_pack(const void* w_bf16, int rows, int cols, int fmt, void* packed,
                       size_t packed_bytes, qmlp_stream_t stream);
int qmlp_quantize_pack_info(const void* packed, int rows, int cols, int fmt, double* max_row_norm,
                            uint32_t* flushed_groups, uint32_t* bad_groups, qmlp_stream_t stream);

/* Inverse of qmlp_pack for bfp8 (lossless for every group that was not flushed): packed ->
 * canonical q/e8.  Used by the on-disk weight cache and the packing audit (the reference audits
 * its packed gate/up the same way, packed_weight_check.cpp:1-37). */
int qmlp_unpack_bfp8(const void* packed, int rows, int cols, void* q, void* e8,
                     qmlp_stream_t stream);

/* Inverse of qmlp_pack for bf4 (same contract as qmlp_unpack_bfp8). */
int qmlp_unpack_bf4(const void* packed, int rows, int cols, void* q, void* e8,
                    qmlp_stream_t stream);

/* Inverse of qmlp_pack for MXFP4: packed -> codes and scales (lossless). */
int qmlp_unpack_mxfp4(const void* packed, int rows, int cols, void* codes, void* scales,
                      qmlp_stream_t stream);

/* Dequantises a packed matrix to fp32 [rows, cols] with the same in-register routine the GEMM
 * kernels use.  Diagnostic/audit use. */
int qmlp_dequant_packed(const void* packed, int rows, int cols, int fmt, float* out,
                        qmlp_stream_t stream);

/* ---------------------------------------------------------------- forward (hot path)
 *
 * Replaces Qwen36MLP.forward(x) (docker/qwen-c2-graft/graft/mlp.py:402-423) and, at M = 16, the
 * reference's fused route FusedT16Arm.forward (scripts/ci/fused_t16_scope.py:45-76):
 * FusedProjection (scripts/ci/fused_1d.py:123-196) + down linear (fused_t16_scope.py:64-67);
 * the residual add of Qwen36DecoderLayer.forward (layer.py:357) is fused when residual != null.
 *
 *   x        bf16 [M, H] row-major
 *   wg, wu   packed [I, H] (gate_proj, up_proj); wd packed [H, I] (down_proj); all in fmt, except
 *            that fmt == QMLP_FMT_BF4 takes wd packed QMLP_FMT_BFP8
 *   residual bf16 [M, H] or null
 *   out      bf16 [M, H]; may alias residual (each element is read before it is written by the
 *            same thread) but must not alias x
 *   ws       workspace of at least qmlp_workspace_bytes(M, H, I, fmt) bytes, initialised once by
 *            qmlp_workspace_init; the kernels leave it re-usable.  Concurrent forwards need
 *            separate workspaces.
 * Constraints: H and I multiples of 256; 1 <= M <= 65536 and, but for QMLP_FMT_MXFP4,
 * M * max(H, I) < 2^30; pointers 16-byte aligned.
 * M <= 32 uses the weight-streaming kernels; larger M the LDS-tiled matrix-core kernels. */
int qmlp_forward(const void* x, const void* wg, const void* wu, const void* wd,
                 const void* residual, void* out, void* ws, size_t ws_bytes, int M, int H, int I,
                 int fmt, qmlp_stream_t stream);

/* qmlp_forward with options.  flags: QMLP_OUT_F32 -- out is fp32 [M, H] (the fp32 sum
 * residual + y, not rounded); QMLP_RESIDUAL_F32 -- residual is fp32 [M, H] (an fp32 residual
 * stream).  qmlp_forward(...) == qmlp_forward_ex(..., 0, stream). */
#define QMLP_OUT_F32 1
#define QMLP_RESIDUAL_F32 2
int qmlp_forward_ex(const void* x, const void* wg, const void* wu, const void* wd,
                    const void* residual, void* out, void* ws, size_t ws_bytes, int M, int H, int I,
                    int fmt, int flags, qmlp_stream_t stream);

/* The decoder's feed-forward half with its RMSNorm prologue:
 *
 *   out = h + down( silu(gate(n)) * up(n) ),   n = h / sqrt(mean(h^2) + eps) * (1 + norm_w)
 *
 * (the zero-centred RMSNorm, mean over H).  Replaces ff_input = self.ffn_norm(h);
 * ff_output = self.feed_forward.forward(ff_input); output = ttnn.add(h, ff_output)
 * (docker/qwen-c2-graft/graft/layer.py:352-357; the norm is the framework RMSNorm with
 * add_unit_offset, layer.py:110-112,228-237).
 *   h       bf16 [M, H], the pre-norm hidden state (also the residual)
 *   norm_w  bf16 [H]
 *   out     bf16 [M, H] (fp32 with QMLP_OUT_F32); may equal h (in-place residual update)
 * Other arguments and constraints as qmlp_forward_ex (QMLP_RESIDUAL_F32 is not accepted).  n is
 * rounded to bf16, as the reference's separate norm writes it.  The norm is one pass over h before the
 * projections; with block-float weights and M > 32 the same pass converts n to fp16. */
int qmlp_forward_rmsnorm(const void* h, const void* norm_w, float eps, const void* wg, const void* wu,
                         const void* wd, void* out, void* ws, size_t ws_bytes, int M, int H, int I,
                         int fmt, int flags, qmlp_stream_t stream);

/* ---------------------------------------------------------------- MXFP4 operators
 *
 * The pieces of the QMLP_FMT_MXFP4 forward as calls of their own, for any sizes: rows M (or N) from
 * 1, K a multiple of 32.  A packed activation matrix has the weights' packed layout
 * (qmlp_packed_bytes(M, K, QMLP_FMT_MXFP4) bytes, without a trailer) and feeds any number of products.
 *
 * The quantisation of a block: its scale is the binade of its largest magnitude less 2, at least
 * 2^-126, so that the largest value lands in [4, 8); values are rounded half to even and saturate at
 * 6.  A block with an infinity or a NaN becomes NaN as a whole (scale byte 255), and so does every
 * output of its row. */
#define QMLP_X_BF16 0
#define QMLP_X_F16 1
#define QMLP_X_F32 2
#define QMLP_X_MXFP4 3 /* already packed: x_stride is not used */
#define QMLP_OUT_MXFP4 4 /* flag of qmlp_mx_swiglu: out is a packed activation matrix [M, N] */

/* x [rows, cols] (x_type BF16, F16 or F32; x_stride elements from row to row, a multiple of 16 bytes)
 * -> packed activation matrix.  Only the given rows are written. */
int qmlp_mx_quantize(const void* x, int x_type, int64_t x_stride, int rows, int cols, void* packed,
                     size_t packed_bytes, qmlp_stream_t stream);

/* The same behind the decoder's zero-centred RMSNorm: n = bf16(h / sqrt(mean(h^2) + eps) * (1 + norm_w)),
 * h bf16 (layer.py:110-112,352-353). */
int qmlp_mx_quantize_rmsnorm(const void* h, int64_t h_stride, const void* norm_w, float eps, int rows,
                             int cols, void* packed, size_t packed_bytes, qmlp_stream_t stream);

/* Packed matrix -> bf16 (out_type QMLP_X_BF16) or fp32 (QMLP_X_F32) [rows, cols], exactly; magnitudes
 * from 2^128 on (scales of 253 and 254 in packed checkpoints) become infinities. */
int qmlp_mx_dequantize(const void* packed, int rows, int cols, void* out, int out_type,
                       qmlp_stream_t stream);

/* out[M, N] = x W^T (+ residual): x of any x_type, quantised in the call unless it is QMLP_X_MXFP4; w
 * packed [N, K].  flags: QMLP_OUT_F32, QMLP_RESIDUAL_F32.  out may be the residual itself (of the same
 * dtype) and must not overlap anything else.  ws: qmlp_mx_workspace_bytes(M, N, K, x_type) bytes that may
 * hold anything (nothing to initialise), null where that is 0; calls that run at the same time need
 * separate ones. */
int qmlp_mx_linear(const void* x, int x_type, int64_t x_stride, const void* w, const void* residual,
                   void* out, void* ws, size_t ws_bytes, int M, int N, int K, int flags,
                   qmlp_stream_t stream);

/* out[M, N] = silu(x Wg^T) * (x Wu^T), the gate/up pair of the block (FusedProjection,
 * scripts/ci/fused_1d.py:123-196).  flags: QMLP_OUT_F32 or QMLP_OUT_MXFP4 (N a multiple of 256; quantised
 * from the fp32 values). */
int qmlp_mx_swiglu(const void* x, int x_type, int64_t x_stride, const void* wg, const void* wu, void* out,
                   void* ws, size_t ws_bytes, int M, int N, int K, int flags, qmlp_stream_t stream);

/* Workspace bytes of the two products (host only); never shrinks as M grows.  0 where none is needed
 * (packed x up to 32 tokens, up to four tokens that the product quantises itself), and for sizes out of
 * range, which the product refuses. */
size_t qmlp_mx_workspace_bytes(int M, int N, int K, int x_type);

/* ---------------------------------------------------------------- 8-bit activations, 4-bit weights
 *
 * The products of the section above with the activations in 8 bits: MXINT8, 32 consecutive K values
 * share a power-of-two scale and each is an integer q in -127..127.  A block whose largest magnitude
 * lies in [2^E, 2^(E+1)) has the step 2^(E-6), with E kept in [-120, 126]; values are rounded half to
 * even, magnitudes beyond 127 steps become 127; a block with an infinity or a NaN becomes NaN as a whole,
 * and so does every output of its row.  The weights are packed QMLP_FMT_MXFP4.  The products and their
 * sums are as exact as those of two 4-bit operands.  A packed activation matrix takes
 * qmlp_mxint8_bytes(rows, cols) bytes (8.25 bits a value) and feeds any number of products. */
#define QMLP_X_MXINT8 4  /* a packed MXINT8 matrix, as x_type of the qmlp_w4a8_* products */
#define QMLP_OUT_MXINT8 8 /* flag of qmlp_w4a8_swiglu: out is a packed MXINT8 matrix [M, N] */

/* Bytes of a packed MXINT8 matrix (host only); 0 for sizes that are not supported (cols not a multiple
 * of 32). */
size_t qmlp_mxint8_bytes(int rows, int cols);

/* x [rows, cols] (x_type BF16, F16 or F32, as for qmlp_mx_quantize) -> packed. */
int qmlp_mxint8_quantize(const void* x, int x_type, int64_t x_stride, int rows, int cols, void* packed,
                         size_t packed_bytes, qmlp_stream_t stream);

/* Packed -> bf16 or fp32 [rows, cols] (out_type QMLP_X_BF16 or QMLP_X_F32), exactly. */
int qmlp_mxint8_dequantize(const void* packed, int rows, int cols, void* out, int out_type, qmlp_stream_t stream);

/* Packed -> the integers (int8 [rows, cols]) and scale bytes E + 127 (uint8 [rows, cols/32]; 255: not a
 * number). */
int qmlp_mxint8_unpack(const void* packed, int rows, int cols, void* q, void* scales, qmlp_stream_t stream);

/* The residual's addition and the decoder's zero-centred RMSNorm of the sum, in one pass
 * (layer.py:352-357 with the addition in front):
 *
 *   h = residual + x,   n = bf16(h / sqrt(mean(h^2) + eps) * (1 + norm_w)),   packed = MXINT8(n)
 *
 *   x         bf16 or fp32 [rows, cols]; residual: bf16 or fp32, or null (then h must be null, and the
 *             norm is that of x)
 *   norm_w    bf16 [cols]
 *   h         [rows, cols] of the residual's type, to which the sum is rounded before the norm; may be the
 *             residual itself (with its stride)
 *   n         bf16 [rows, cols] contiguous, or null; packed: a packed MXINT8 matrix, or null; not both null
 * Strides count elements from row to row and are multiples of 16 bytes.  Outputs must not overlap each other
 * or (but for h on the residual) an input. */
int qmlp_add_rmsnorm(const void* x, int x_type, int64_t x_stride, const void* residual, int residual_type,
                     int64_t residual_stride, const void* norm_w, float eps, int rows, int cols, void* h,
                     int64_t h_stride, void* n, void* packed, size_t packed_bytes, qmlp_stream_t stream);

/* qmlp_mx_linear with 8-bit activations: x BF16, F16 or F32 rows, quantised in the call, or QMLP_X_MXINT8. */
int qmlp_w4a8_linear(const void* x, int x_type, int64_t x_stride, const void* w, const void* residual,
                     void* out, void* ws, size_t ws_bytes, int M, int N, int K, int flags,
                     qmlp_stream_t stream);

/* out[M, N] = silu(x Wg^T + gate_add) * (x Wu^T + up_add): qmlp_mx_swiglu with 8-bit activations.  gate_add
 * and up_add: fp32 [M, N] or null, what low-rank adapters add to the projections.  flags: QMLP_OUT_F32 or
 * QMLP_OUT_MXINT8 (N a multiple of 256; quantised from the fp32 values). */
int qmlp_w4a8_swiglu(const void* x, int x_type, int64_t x_stride, const void* wg, const void* wu,
                     const float* gate_add, const float* up_add, void* out, void* ws, size_t ws_bytes, int M,
                     int N, int K, int flags, qmlp_stream_t stream);

/* Workspace bytes of the two products (host only), like qmlp_mx_workspace_bytes; it may hold anything. */
size_t qmlp_w4a8_workspace_bytes(int M, int N, int K, int x_type);

/* ---------------------------------------------------------------- low-rank adapters
 *
 * What the adapters of a batch's requests add beside one shared projection:
 *
 *   out[m] = base[m] + s_a B_a (A_a x[m]),   a = ids[m];  A_a [rank, K], B_a [N, rank], s_a a number
 *
 * for any number of adapters from 1 to 1024 of ranks from 1 to 128, which may differ.  A token whose id is
 * outside [0, adapters) has none (out[m] = base[m]).
 *
 * Layouts (ranks padded with zeros to units of 16 in a, of 32 in b):
 *   a     [unit][K / 32][64][8] 16-bit values: lane l of a K-step holds rank l % 16 of the unit, K values
 *         8 (l / 16)..; adapter after adapter
 *   b     per adapter [N / 64, rounded up][unit][4][64][8]: in part f lane l holds ranks 8 (l / 16).. of the
 *         unit for feature 16 f + l % 16 of the block (zeros behind N); adapter after adapter
 *   meta  int32 [adapters][4]: {rank, units of a in the adapters before, the bits of s_a (fp32), units of b
 *         before}
 *
 * A plan groups a batch's tokens by adapter; it serves every projection with the same adapter numbers (all of a
 * model's layers) until the tokens' adapters change. */
size_t qmlp_lora_plan_bytes(int M, int adapters); /* host only; 0 for sizes out of range */
int qmlp_lora_plan(const int32_t* ids, int M, int adapters, void* plan, size_t plan_bytes, qmlp_stream_t stream);

/* x: bf16 or fp16 [M, K] (x_type; x_stride elements from row to row, a multiple of 16 bytes), the type of a and
 * b; plan: qmlp_lora_plan's for the same M and number of adapters (with another one nothing is written);
 * base: bf16 or fp32 [M, N] (QMLP_RESIDUAL_F32) or null; out: bf16 or fp32 [M, N] (QMLP_OUT_F32), may be base of
 * the same type.  Sums are fp32, rounded once.  ws: qmlp_lora_workspace_bytes(M, K, max_rank) bytes that may hold
 * anything; calls that run at the same time need separate ones. */
int qmlp_lora_linear(const void* x, int x_type, int64_t x_stride, const void* a, const void* b, const void* meta,
                     int adapters, int max_rank, const void* plan, const void* base, void* out, void* ws,
                     size_t ws_bytes, int M, int N, int K, int flags, qmlp_stream_t stream);
size_t qmlp_lora_workspace_bytes(int M, int K, int max_rank); /* host only; never shrinks as M grows */

/* Workspace bytes needed by qmlp_forward for these sizes (host only, no GPU needed).  The size
 * never decreases as M grows, so a workspace sized for M serves every call with fewer tokens, and
 * one workspace serves calls of different shapes as long as it is large enough for each. */
size_t qmlp_workspace_bytes(int M, int H, int I, int fmt);

/* The first QMLP_WS_COUNTER_BYTES bytes of every workspace hold arrival counters, at the same
 * place for every shape.  They must read zero when a forward starts, and every forward leaves them
 * zero.  The rest of the workspace may hold anything when a forward starts. */
#define QMLP_WS_COUNTER_BYTES 524288

/* Zero-fills the workspace with a kernel (not a memset node, so it may be graph-captured). */
int qmlp_workspace_init(void* ws, size_t ws_bytes, qmlp_stream_t stream);

/* qmlp_forward_ex without a workspace argument.  No counterpart in the reference: this entry point
 * is for callers that cannot allocate device memory (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc).  The workspace is a QMLP_SCRATCH_BYTES array of device
 * memory inside the library, one per GPU, held until the process ends; the call allocates and
 * frees nothing.  It serves every call whose qmlp_workspace_bytes(M, H, I, fmt) fits, e.g. M <= 32
 * at H = 5120, I = 17408; larger calls fail with QMLP_E_WORKSPACE.  The array starts zeroed (it
 * is loaded with the library's code object), and every forward leaves its arrival counters at
 * zero.  The first call on a device looks up the array's address (hipGetSymbolAddress) and must
 * be made outside graph capture: a first call on a capturing stream fails with QMLP_E_LAUNCH;
 * later calls may be captured.  Every call on one GPU shares that GPU's array: calls that overlap
 * on one GPU (several streams or host threads) race and must be serialised by the caller.
 * Arguments, constraints and results as qmlp_forward_ex. */
#define QMLP_SCRATCH_BYTES 33554432
int qmlp_forward_noalloc(const void* x, const void* wg, const void* wu, const void* wd,
                         const void* residual, void* out, int M, int H, int I, int fmt, int flags,
                         qmlp_stream_t stream);

/* ---------------------------------------------------------------- profiling (host only)
 *
 * Per-kernel timing of the forward pass, the counterpart of the reference's per-op signposts
 * (docker/qwen-c2-graft/graft/layer.py:18-90).  When n == 4, every later qmlp_forward on this host
 * thread launches its gate/up kernel with events[0] / events[1] as the start / stop events of
 * hipExtLaunchKernel and its down kernel with events[2] / events[3] (hipEvent_t handles): each
 * pair then holds the timestamps of that dispatch itself, and no marker packets are inserted
 * between the kernels.  n == 0 turns timing off.  Kernels outside the two projections (the
 * RMSNorm pass, the prefill's activation prep) are not timed. */
int qmlp_set_profile_events(void* const* events, int n);

/* ---------------------------------------------------------------- planning (host only)
 *
 * Work split of the M <= 32 stream-K kernel (the fallback where qmlp_plan_split finds no split)
 * for one projection: `rows` output rows (multiple of 16) over K (multiple of 256) on `num_cus`
 * compute units.  Fills out[0..1] =
 * {workgroups, tiles one wave may touch}.  Exposed so the coverage of the split can be tested
 * without a GPU, like the reference's worker-to-pair mapping tests
 * (scripts/ci/test_fused_1d.py:71-79). */
int qmlp_plan_stream(int rows, int K, int num_cus, int* out2);

/* Work split of the many-token kernel (M > 32) for one projection of an MLP of `fmt` weights (down
 * != 0: the down projection, [H, I]; else the gate/up pair) on `num_cus` compute units.  Fills
 * out[0..7] = {features per tile, tokens per tile, tiles, leading tiles that run whole, K pieces of
 * each other tile (1: none is split), blocks launched, bytes of one piece's partial tile, bytes the
 * workspace holds for the pieces}. */
int qmlp_plan_tiles(int M, int H, int I, int fmt, int down, int num_cus, int* out8);

/* Work split of the M <= 32 weight-streaming kernel for one projection with `nmat` matrices
 * (2 = gate/up, 1 = down) at M tokens (1..32; 17..32 run as two groups of 16): the (16-row tile
 * x 256-K superblock) grid cut into tile groups x K splits, split q covering superblocks
 * [q*C/S, (q+1)*C/S) of C = K/256.  Fills out[0..5] = {workgroups, tiles per group, K splits,
 * superblocks of the longest split, groups, tiles one wave may touch}. */
int qmlp_plan_split(int rows, int K, int nmat, int M, int num_cus, int* out6);

/* How an MXFP4 product of M tokens, N output and K input features and `nmat` matrices (2 = gate/up)
 * runs on `num_cus` compute units.  Fills out[0..4] = {kernel, pieces of the K range, workgroups, KB of
 * partial tiles, 1 where the kernel also quantises unpacked rows}.  Kernels: 0 a workgroup of four waves
 * per 32 features and 32 tokens, 1 the same with twice the loads under way, 2 of eight waves, 3 per 32
 * features and 64 tokens, 3 + h tiles of 256 features (of both matrices together) x 64 h tokens. */
int qmlp_mx_plan(int M, int N, int K, int nmat, int num_cus, int* out5);

/* The same for the products with 8-bit activations: 0 to 3 as there with one unit's loads under way (1: two), 3 + h
 * for h = 1, 2, of which full rounds may run whole and the rest in pieces of the K range, 8 the kernel of up to 16
 * tokens. */
int qmlp_w4a8_plan(int M, int N, int K, int nmat, int num_cus, int* out5);

/* How qmlp_lora_linear runs for these sizes (host only; adapters: those loaded): out5 = {launches; units of 16 tokens of
 * a tile; the most units of 16 ranks that the kernels are made for; pieces of the K range; the most that K would give}. */
int qmlp_lora_path(int M, int N, int K, int adapters, int max_rank, int num_cus, int* out5);

#ifdef __cplusplus
}
#endif

#endif /* QWEN_MLP_H */
