/*
 * weightferry.h -- C ABI of the MI355X (gfx950) quantized-weight hot path.
 *
 * One shared library, libweightferry_hip.so, built from comfyui-weightferry_amd/csrc/. Plain pointers and sizes
 * only; every device pointer is memory the caller allocated (the library never allocates or frees device memory
 * on these paths). `stream` is a hipStream_t (NULL = the default stream); every call is asynchronous on it and
 * never synchronises the host.
 *
 * Return codes: WF_OK (0) on success; WF_EUNSUPPORTED (-2) when the call is "not my case" (the reference's
 * Python returns None there and the host application's own code runs); WF_EINVAL (-1) for malformed arguments;
 * WF_EHIP (-3) when a HIP runtime call failed. wf_last_error() gives a thread-local message for the last failure
 * on the calling thread.
 *
 * Dtype codes follow enhancers/gguf_dequant.py:58 of the reference: 0 float16, 1 bfloat16, 2 float32.
 * GGML type ids follow enhancers/gguf_dequant.py:52-56: 2 Q4_0, 3 Q4_1, 6 Q5_0, 7 Q5_1, 8 Q8_0, 10 Q2_K, 11 Q3_K,
 * 12 Q4_K, 13 Q5_K, 14 Q6_K.
 */
#ifndef WEIGHTFERRY_H
#define WEIGHTFERRY_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define WF_OK 0
#define WF_EINVAL (-1)
#define WF_EUNSUPPORTED (-2)
#define WF_EHIP (-3)

#define WF_F16 0
#define WF_BF16 1
#define WF_F32 2

/* ABI version (bumped on any signature change) and the last error message of the calling thread. */
int wf_abi_version(void);
const char* wf_last_error(void);

/* ---------------------------------------------------------------------------------------------- dequantisation
 * Replaces the Triton launches of `dequantize` / `_dequantize_k` (enhancers/gguf_dequant.py:277-326; kernels
 * `_deq` :136-167 and `_deq_k` :188-256). `src` holds src_bytes of GGUF blocks of type `qtype`; `out` receives
 * n_values values of dtype out_dt, each computed with the reference's rounding chain in the dequant dtype mid_dt.
 * WF_EUNSUPPORTED when qtype / dtypes are not handled or src_bytes does not hold exactly n_values values (the
 * reference returns None there, :280-286,312-320), or when src / out are not 16-byte aligned. */
int wf_dequant(const void* src, int64_t src_bytes, int qtype, int mid_dt, int out_dt, void* out, int64_t n_values,
               void* stream);

/* LoRA add on a GGUF weight: replaces the Triton kernel `_deq_add` (enhancers/gguf_dequant.py:99-133) as
 * `_add_loras` launches it once per LoRA (:387-409). out[i] = OUT(w + OUT(diff[i] * scale)) for i < n_values, the
 * product, the sum and each rounding on their own; w is the dequantisation of `src` exactly as wf_dequant gives it
 * (the first LoRA, DEQ on) when src is not NULL, else the value already in out (a later LoRA; qtype, src_bytes
 * and mid_dt are then ignored). diff: float32 [n_values], comfy's up @ down of one LoRA; scale = strength *
 * alpha / rank. The reference dequantises a K-quant by its own kernel and adds every LoRA afterwards; here the
 * first add is fused into the K-quant dequantisation too (the same values). out and diff 16-byte aligned. */
int wf_dequant_add(const void* src, int64_t src_bytes, int qtype, int mid_dt, int out_dt, const float* diff,
                   float scale, void* out, int64_t n_values, void* stream);

/* The same add with the difference computed inside the kernel from the LoRA's factors: diff = up @ down in float32
 * (up [n_out, rank] of dtype up_dt, down [rank, n_in] of dtype down_dt, both row-major on the device; float16 and
 * bfloat16 are widened exactly), out [n_out, n_in]. src as in wf_dequant_add: NULL adds onto the values in out.
 * rank 1..192; rows are whole blocks of qtype (a multiple of 8 values without src); out 16-byte aligned, down aligned
 * to two of its values. */
int wf_dequant_lora(const void* src, int64_t src_bytes, int qtype, int mid_dt, int out_dt, const void* up, int up_dt,
                    const void* down, int down_dt, int64_t rank, float scale, void* out, int64_t n_out, int64_t n_in,
                    void* stream);

/* ---------------------------------------------------------------------------------------------- int8 W8A8 path
 * Per-row int8 quantisation of bf16 activations: replaces the Triton `_quant_row` with PRE_NONE
 * (enhancers/fused_kernels.py:137-174, launched at enhancers/fused_int8.py:172-176) and kitchen's
 * quantize_int8_rowwise_convrot64 (enhancers/fused_int8.py:178-181). mode 0: plain per-token (K % 16 == 0,
 * K <= 32768); mode 1: ConvRot 256-groups (K % 256 == 0, K <= 32768). x: bf16 [M, K] row-major; xq: int8 [M, K];
 * xs: float32 [M]. x and xq 16-byte aligned. */
int wf_quant_rows_i8(const void* x_bf16, int64_t M, int64_t K, int mode, int8_t* xq, float* xs, void* stream);

/* The ConvRot quantisation (mode 1 above) with an operation applied to each value first: replaces the Triton
 * `_quant_row` with PRE 1..3 (enhancers/fused_kernels.py:137-163) as `_quantise_pre` launches it for a pending input
 * (enhancers/fused_int8.py:60-75). pre 0: none; 1 GELU: y = table[bits(x)], s_bf16 = torch's GELU of all 65536 bf16
 * values (:94-105); 2 MOD: y = bf16(bf16(x * s1) + shift) with s_bf16 = s1 = 1 + scale and shift_bf16 = shift, both
 * bf16 [M / rows_per_group, K], row r using group r / rows_per_group (:28-39); 3 LNMOD: LayerNorm without affine
 * first -- mean and variance by the reference's Welford order (:84-136), rstd = 1 / sqrt(var + eps) correctly rounded
 * where the reference uses the NVIDIA approximation rsqrt.approx.f32 -- rounded to bf16, then MOD. K % 256 == 0,
 * K <= 32768 (LNMOD: K % 512 == 0); s / shift 16-byte aligned for MOD / LNMOD. */
int wf_quant_rows_i8_pre(const void* x_bf16, int64_t M, int64_t K, int pre, const void* s_bf16, const void* shift_bf16,
                         int64_t rows_per_group, float eps, int8_t* xq, float* xs, void* stream);

/* out[m, n] = OUT((float(acc[m, n]) * xs[m]) * ws[n] (+ bias[n])), acc = sum_k xq[m, k] * wq[n, k] exactly in
 * int32: replaces kitchen's cutlass_int8_dequant (enhancers/fused_int8.py:191-206; the reference returns None and
 * falls back where this returns WF_EUNSUPPORTED). wq is [N, K] (row = output channel); bias (nullable) has dtype
 * out_dt; out_dt is WF_BF16 or WF_F16. K % 16 == 0, xq / wq 16-byte aligned. */
int wf_linear_i8(const int8_t* xq, const int8_t* wq, const float* xs, const float* ws, const void* bias, void* out,
                 int out_dt, int64_t M, int64_t N, int64_t K, void* stream);

/* out = bf16(resid + gate[m / rows_per_group] * bf16((float(acc) * xs[m]) * ws[n])): wf_linear_i8's bf16 output
 * followed by torch.addcmul(resid, gate, out) on bf16 tensors (the product exact in float32, the sum rounded once
 * to float32, then to bf16) -- replaces kitchen's cutlass_int8_dequant_residual, which the reference states gives
 * those bits (enhancers/fused_int8.py:212-268: x_res + gate * linear(x) per (batch, frame) group of rows;
 * enhancers/fused_block.py:24-26). gate: bf16 [M / rows_per_group, N]; resid, out: bf16 [M, N]. */
int wf_linear_i8_residual(const int8_t* xq, const int8_t* wq, const float* xs, const float* ws, const void* gate_bf16,
                          const void* resid_bf16, void* out_bf16, int64_t M, int64_t N, int64_t K,
                          int64_t rows_per_group, void* stream);

/* Either form with a workspace, in which a product too small to fill the chip runs as K slices whose int32 sums are
 * added afterwards (the same bits): gate and resid NULL for the plain form, both set for the residual one (then bias is
 * NULL and out_dt WF_BF16). wf_linear_i8_workspace gives the bytes for a shape (0: none needed); the workspace is
 * 256-byte aligned, need not be cleared and is free again when the call's work on the stream is done. */
int wf_linear_i8_workspace(int64_t M, int64_t N, int64_t K, int64_t* bytes);
int wf_linear_i8_ws(const int8_t* xq, const int8_t* wq, const float* xs, const float* ws, const void* bias,
                    const void* gate_bf16, const void* resid_bf16, void* out, int out_dt, int64_t M, int64_t N,
                    int64_t K, int64_t rows_per_group, void* workspace, int64_t workspace_bytes, void* stream);

/* How a product runs when it may use a workspace of workspace_bytes (0: wf_linear_i8, wf_linear_i8_residual; INT64_MAX:
 * wf_linear_i8_ws). tile_rows 0: the kernel for K that is not a multiple of 64. whole_ns is the modelled GPU time without
 * slices, 0 where nothing is modelled (then there are no slices): a caller bound by its own thread can do without them. */
typedef struct {
    int32_t tile_rows, tile_columns, slices;
    int64_t workspace_bytes, whole_ns;
} wf_i8_plan;
int wf_linear_i8_plan(int64_t M, int64_t N, int64_t K, int64_t workspace_bytes, wf_i8_plan* plan);

/* ------------------------------------------------------------------------------- fused dequant + bf16 GEMM
 * y[m, n] = bf16(sum_k x[m, k] * W[n, k] (+ bias[n])) with W given as GGUF K-quant blocks (qtype 12 Q4_K, 13 Q5_K, 14
 * Q6_K; [N, K] row-major in 256-value super-blocks, wq_bytes = N * K / 256 * block bytes; also qtype 8 Q8_0, 34 bytes
 * per 32 values, at 1-512 rows only, WF_EUNSUPPORTED elsewhere; its panels take 64 rows, and wf_linear_gguf_ws and
 * wf_linear_gguf_noalloc give it the panel form at the K-quants' rows) and dequantised inside the kernel exactly as
 * wf_dequant does with dequant dtype mid_dt and output bf16; float32 accumulation. No reference function does this in
 * one step: it replaces `dequantize` (enhancers/gguf_dequant.py:296-326) followed by ComfyUI-GGUF's
 * torch.nn.functional.linear on the bf16 weight. x: bf16 [M, K], 16-byte aligned; bias: bf16 [N] or NULL; out: bf16
 * [M, N]. K % 256 == 0, K <= 1048576. M <= 64 runs the few-rows forms (the weight streamed once; at 1-3 rows of N <
 * 8192, Q6_K and Q8_0 1-4 rows of N < 16384: workgroups of whole 4-row quads), 65-512 rows the panel form, larger M
 * the tiled form (256 x 320 tiles; Q6_K from 1024 rows 512 x 160). */
int wf_linear_gguf(const void* x_bf16, int64_t M, int64_t K, const void* wq, int64_t wq_bytes, int qtype, int64_t N,
                   const void* bias_bf16, void* out_bf16, int mid_dt, void* stream);

/* wf_linear_gguf with a caller-provided workspace, for the same reference call site (enhancers/gguf_dequant.py:
 * 296-326 followed by ComfyUI-GGUF's F.linear). A narrow, deep product (N <= 2048, K >= 8192, K >= 2 N) with 1 <= M <=
 * 8 rows is split along K over many more workgroups than weight rows allow: each writes float32 partial sums into the
 * workspace, and the last workgroup of each column tile adds them in a fixed order (the result is the same on every
 * run). Workspace: 256-byte aligned, at least the bytes wf_linear_gguf_workspace gives; its first 16 KiB are counters
 * that must be zero on entry and are zero again when the call has run, whatever its shape (a workspace cleared once
 * can be reused by later calls of any shape on the same stream; calls that overlap on one workspace race). With 33-512
 * rows, and with 17-32 rows of a deep product (K >= 2 N), the panel form splits K into slices (at least two
 * super-blocks each), enough to give the chip 256 workgroups: each slice writes float32 partial sums into the
 * workspace past the split form's 16 KiB of counters, which it leaves untouched (16 KiB + S * M * N * 4 bytes), and a
 * second kernel adds them in slice order; up to 64 rows only when K gives more than one slice.
 * wf_linear_gguf_workspace does not know the format and gives the largest need over them. Any other shape does not use
 * the workspace (workspace may be NULL) and is wf_linear_gguf. */
int wf_linear_gguf_workspace(int64_t M, int64_t N, int64_t K, int64_t* bytes);
int wf_linear_gguf_ws(const void* x_bf16, int64_t M, int64_t K, const void* wq, int64_t wq_bytes, int qtype, int64_t N,
                      const void* bias_bf16, void* out_bf16, int mid_dt, void* workspace, int64_t workspace_bytes,
                      void* stream);

/* wf_linear_gguf_ws without the workspace argument: allocates nothing. No counterpart in the reference; it is for
 * callers that cannot allocate device memory (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc). The split form's counters and partial sums live in a 16 MiB array the library holds on each GPU
 * it runs on until the process ends; the counters are cleared by a small kernel on `stream` at the start of each call
 * (no memset). A shape that needs more than 16 MiB there returns WF_EUNSUPPORTED with a message. The panel form
 * (the rows of wf_linear_gguf_ws) takes as many K slices as fit the array past the counters (one, and no scratch, at
 * worst; up to 64
 * rows one slice leaves the call to the few-rows kernel). Every call on a GPU shares
 * that GPU's array: calls that overlap on one GPU (on different streams or threads) race. */
int wf_linear_gguf_noalloc(const void* x_bf16, int64_t M, int64_t K, const void* wq, int64_t wq_bytes, int qtype,
                           int64_t N, const void* bias_bf16, void* out_bf16, int mid_dt, void* stream);

/* y[m, n] = bf16(sum_k x[m, k] * w[n, k] (+ bias[n])), float32 accumulation: the GEMM of the two-step flow, after
 * wf_dequant -- replaces ComfyUI-GGUF's torch.nn.functional.linear on the weight that `dequantize`
 * (enhancers/gguf_dequant.py:296-326) returns. x: bf16 [M, K], w: bf16 [N, K], both 16-byte aligned; bias: bf16 [N]
 * or NULL; out: bf16 [M, N]. K % 64 == 0 and M * K, N * K < 2^30, else WF_EUNSUPPORTED (the caller's own GEMM runs).
 * Tiles of 256 x 320, 256 x 256, 256 x 128 or 128 x 160 outputs, whichever fills the chip best. */
int wf_linear_bf16(const void* x_bf16, const void* w_bf16, const void* bias_bf16, void* out_bf16, int64_t M, int64_t N,
                   int64_t K, void* stream);

/* -------------------------------------------------------------------------------- a training step's operators
 * No reference counterpart: the reference runs its models only; these fine-tune a block next to the inference path.
 *
 * LayerNorm over rows of K <= 32768 values of type dt: y = (x - mean) rstd s + b, s = w (plus_one 0) or 1 + w, each sum in
 * float32. w and b (either may be NULL) are [M / rows_per_group, K] of type param_dt (dt or WF_F32), row r using row r /
 * rows_per_group: rows_per_group = M for affine weights, the rows of one batch entry for a DiT block's modulation. x: M
 * rows ldx values apart; y: [M, K]; stats (may be NULL): float32 [M, 2], mean and rstd, what the backward pass reads.
 * Pointers need only their values' alignment. At most 65535 groups. */
int wf_layer_norm(const void* x, int64_t ldx, int dt, const void* w, const void* b, int param_dt, int plus_one,
                  int64_t rows_per_group, float eps, void* y, float* stats, int64_t M, int64_t K, void* stream);

/* Its gradients: dx [M, K] of type dt, dw and db [M / rows_per_group, K] of type param_dt; any of the three may be NULL.
 * dy: M rows ldd values apart. The workspace (needed for dw and db: the bytes that wf_layer_norm_bwd_workspace gives, 4-byte
 * aligned) holds partial sums; they are added in a fixed order, so the results are the same on every run. */
int wf_layer_norm_bwd_workspace(int64_t M, int64_t K, int64_t rows_per_group, int dt, int64_t* bytes);
int wf_layer_norm_bwd(const void* x, int64_t ldx, const void* dy, int64_t ldd, int dt, const void* w, int param_dt,
                      int plus_one, int64_t rows_per_group, const float* stats, void* dx, void* dw, void* db, int64_t M,
                      int64_t K, void* workspace, int64_t workspace_bytes, void* stream);

/* The norms after and before two sub-layers with the gated residual between them, rows of K values of type dt, at most 32768
 * bytes: r = scale x + gate post_weight n(h), y = norm(r) s + bias, s = weight (plus_one 0) or 1 + weight. n: post, 0 nothing, 1
 * RMS, h / sqrt(mean h^2 + eps), 2 LayerNorm; norm: 1 or 2. post_weight: [K]; gate: [gate_groups, K]; weight, bias:
 * [weight_groups, K], gate_groups and weight_groups 1 or groups: the M rows are `groups` runs of consecutive rows, each with a row of
 * those. Any of the four may be NULL; each is of type dt or WF_F32 (weight and bias of one). h may be NULL (r = scale x), and r.
 * x, h: rows x_row, h_row values apart; r, y: [M, K]; y comes from r before its rounding. stats (may be NULL): float32 [M, 4],
 * mean (0 for RMS) and reciprocal root of h's norm and of r's, what the backward pass reads.
 * wf_block_norm_bwd: dx and dh [M, K] of type dt, the parameters' gradients of their types, for the gradients dr of r and dy of
 * y (either may be NULL); any output may be NULL; bias is not read. The workspace (for as many parameters' gradients, `sums`, as are
 * wanted; 4-byte aligned) holds partial sums, added in a fixed order. */
typedef struct {
    int32_t dt, post, norm, plus_one;
    int32_t post_weight_dt, gate_dt, weight_dt;
    float scale, eps;
    int64_t groups, gate_groups, weight_groups;
} wf_block_norm;
int wf_block_norm_fwd(const wf_block_norm* q, const void* x, int64_t x_row, const void* h, int64_t h_row, const void* post_weight,
                      const void* gate, const void* weight, const void* bias, void* r, void* y, float* stats, int64_t M, int64_t K,
                      void* stream);
int wf_block_norm_bwd_workspace(const wf_block_norm* q, int64_t M, int64_t K, int sums, int64_t* bytes);
int wf_block_norm_bwd(const wf_block_norm* q, const void* x, int64_t x_row, const void* h, int64_t h_row, const void* post_weight,
                      const void* gate, const void* weight, const void* dr, int64_t dr_row, const void* dy, int64_t dy_row,
                      const float* stats, void* dx, void* dh, void* dpost_weight, void* dgate, void* dweight, void* dbias, int64_t M,
                      int64_t K, void* workspace, int64_t workspace_bytes, void* stream);

/* y[m, n] = resid[m, n] + gate[m / rows_per_group, n] * act(sum_k x[m, k] * w[n, k] + bias[n]) in dt (WF_BF16 or WF_F16),
 * float32 accumulation, one rounding. act: 0 none, 1 GELU (erf), 2 GELU (tanh), 3 SiLU, 4 ReLU. bias, gate, resid may be
 * NULL; bias and gate have type dt or WF_F32 (bias_dt, gate_dt). An operand's value (r, k) is at r * row + k * col, so
 * transposed views need no copy by the caller; resid's rows are resid_row values apart; y is [M, N]. h (may be NULL): the
 * sums with the bias, [M, N], rounded to dt, what wf_dense_bwd reads (kept finite). M, N <= 2^24, K <= 2^20.
 * The workspace (256-byte aligned, at least the bytes that wf_dense_workspace gives for the same operands; epilogue: 1 with an
 * activation, + 2 where h is kept, + 4 with a gate or resid) holds copies of operands that cannot be loaded as they are, and
 * the float32 partial sums of products that run in slices of K, or with w across K and any such epilogue; it need not be
 * cleared and is free again when the call's work on the stream is done. */
int wf_dense_workspace(const void* x, int64_t x_row, int64_t x_col, const void* w, int64_t w_row, int64_t w_col, int dt,
                       int64_t M, int64_t N, int64_t K, int epilogue, int64_t* bytes);
/* How wf_dense runs such a call, plan[5]: the kernel (0 few rows; tiles: 1 both operands along K, 2 the same with an
 * activation, gate, resid or h in its epilogue, 3 w across K, 4 both across), its tiling (0-7; few rows: 16-row weight tiles a
 * workgroup), slices of K, and how x and w get there (0 as they lie along K, 1 as they lie across, 2 and 3 copied in that
 * order, 4 copied into rows along K). */
int wf_dense_plan(const void* x, int64_t x_row, int64_t x_col, const void* w, int64_t w_row, int64_t w_col, int dt, int64_t M,
                  int64_t N, int64_t K, int epilogue, int* plan);
int wf_dense(const void* x, int64_t x_row, int64_t x_col, const void* w, int64_t w_row, int64_t w_col, int dt, int64_t M,
             int64_t N, int64_t K, const void* bias, int bias_dt, int act, const void* gate, int gate_dt,
             int64_t rows_per_group, const void* resid, int64_t resid_row, void* y, void* h, void* workspace,
             int64_t workspace_bytes, void* stream);

/* Its backward pass for the gradient dy of y (rows dy_row values apart), h as wf_dense left it (NULL without an activation
 * and dgate): dh = dy gate act'(h) is rounded to dt, then dx = dh . w [M, K], dw = dh^T . x [N, K], dbias = the sum over rows
 * of the unrounded dh (bias_dt), dgate = the sum over each group's rows of dy act(h) (gate_dt); any of the four may be NULL.
 * (resid's gradient is dy.) x: rows x_row values apart; w as in wf_dense. M, N, K <= 2^20, at most 65535 groups. The workspace
 * (256-byte aligned; wf_dense_bwd_workspace for the same operands, gated: whether there is a gate, dx, dw: whether they
 * are wanted, sums: dbias or dgate is) holds dh, partial sums (for both of dbias and dgate) and what the products need. Every
 * sum has a fixed order. */
int wf_dense_bwd_workspace(const void* x, int64_t x_row, const void* w, int64_t w_row, int64_t w_col, const void* dy,
                           int64_t dy_row, int dt, int act, int gated, int64_t rows_per_group, int64_t M, int64_t N,
                           int64_t K, int dx, int dw, int sums, int64_t* bytes);
int wf_dense_bwd(const void* x, int64_t x_row, const void* w, int64_t w_row, int64_t w_col, const void* dy, int64_t dy_row,
                 const void* h, int dt, int act, const void* gate, int gate_dt, int64_t rows_per_group, int64_t M,
                 int64_t N, int64_t K, void* dx, void* dw, void* dbias, int bias_dt, void* dgate, void* workspace,
                 int64_t workspace_bytes, void* stream);

/* The gated feed-forward layer's first half: g, u = the halves of x w^T + bias, y[m, n] = act(g[m, n]) u[m, n] in dt (WF_BF16 or
 * WF_F16), float32 accumulation, one rounding. w: [2 N, K], the gate's rows first; bias (may be NULL): [2 N] of type dt or
 * WF_F32; y: [M, N]; operands and act as in wf_dense. kept (may be NULL): 6 M N bytes, g and u in 24 bits for wf_gated_dense_bwd.
 * M <= 2^20, N <= 2^19, K <= 2^20. wf_gated_dense_plan: the workspace's bytes (256-byte aligned; it need not be cleared) and how
 * such a call runs, plan[5]: 0 few rows, 1 tiles or 2 tiles of rows that start anywhere, the tiling (0-4; 0-1), slices of K, and how x
 * and w get there as in wf_dense_plan. */
int wf_gated_dense_plan(const void* x, int64_t x_row, int64_t x_col, const void* w, int64_t w_row, int64_t w_col, int dt,
                        int64_t M, int64_t N, int64_t K, int keep, int* plan, int64_t* bytes);
int wf_gated_dense(const void* x, int64_t x_row, int64_t x_col, const void* w, int64_t w_row, int64_t w_col, int dt, int64_t M,
                   int64_t N, int64_t K, const void* bias, int bias_dt, int act, void* y, void* kept, void* workspace,
                   int64_t workspace_bytes, void* stream);

/* Its backward pass for the gradient dy of y (rows dy_row values apart): dg = dy u act'(g), du = dy act(g), dh = [dg du] rounded to
 * dt, dx = dh w [M, K], dw = dh^T x [2 N, K], dbias the sums over rows of the unrounded dh [2 N]; any of the three may be NULL. Every
 * sum has a fixed order. WF_F16: where dh's largest finite magnitude is past 65504 or below 2^-8, dh is rounded times a power of two that
 * brings it to 2^14, and the products are multiplied back. */
int wf_gated_dense_bwd_workspace(const void* x, int64_t x_row, const void* w, int64_t w_row, int64_t w_col, int dt, int64_t M,
                                 int64_t N, int64_t K, int dx, int dw, int db, int64_t* bytes);
int wf_gated_dense_bwd(const void* x, int64_t x_row, const void* w, int64_t w_row, int64_t w_col, const void* dy, int64_t dy_row,
                       const void* kept, int dt, int act, int64_t M, int64_t N, int64_t K, void* dx, void* dw, void* dbias,
                       int bias_dt, void* workspace, int64_t workspace_bytes, void* stream);

/* One AdamW step (step >= 1) of `count` tensors of type dt, in place: m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2,
 * p = (1 - lr decay) p - lr / (1 - b1^step) * m / (sqrt(v) / sqrt(1 - b2^step) + eps). table: host memory, read before the
 * call returns: address of the parameter, address of its gradient, values, for each tensor. The moments are flat over all
 * tensors, each starting on a whole block of 256 values, `blocks` in all: bits 32: float32 [blocks * 256], scales unused;
 * bits 8: exp_avg int8, exp_avg_sq uint8 [blocks * 256] with float32 scales [blocks], m = sign(q) (q / 127)^2 s, v = ((q /
 * 255)^2 s)^2, s a block's largest |m| or sqrt(v); a v > 0 keeps a code > 0. Captured into a graph, a replay repeats this
 * step: rates, bias corrections and addresses are the launch's. wf_adamw_values: the float32 values that 8-bit
 * moments stand for. */
int wf_adamw(const int64_t* table, int64_t count, int dt, int bits, void* exp_avg, void* exp_avg_sq, float* avg_scale,
             float* sq_scale, int64_t blocks, int64_t step, double lr, double beta1, double beta2, double eps,
             double weight_decay, void* stream);
int wf_adamw_values(const int8_t* exp_avg, const uint8_t* exp_avg_sq, const float* avg_scale, const float* sq_scale,
                    int64_t blocks, float* avg, float* sq, void* stream);

/* Orthogonalised updates of `count` matrices [rows, cols] of type dt, row-major and contiguous: m = mu m + (1 - mu) g, u = (1 - mu) g + mu
 * m (nesterov) or m, X = u / max(|u|, eps) with the Frobenius norm, `steps` times (1 to 32) X = a X + (b A + c A A) X, A = X X^T; then p =
 * keep p - rate X, in place (p and m). table: host memory, read before the call returns: addresses of p, g and m of each matrix; m
 * (float32) may be 0: u = g. coefficients: a, b, c; WF_EINVAL for ones that take singular values from [0, 1] past 1.9. The shorter side
 * <= 16384, the longer <= 2^20, (rows + 256) (cols + 8) < 2^30. No matrix may be there twice. With a shorter side up to 64 everything
 * is float32 or more; above, the products' operands are float16, for float32 matrices too, and X is off by about 1e-3 of its norm for flat and
 * falling spectra, by up to 4e-3 where few directions hold nearly all of a matrix, 1.5e-2 where two or three entries do (singular values on
 * the polynomial's steep parts). wf_orthogonalize: out = X, table: addresses of out, g and 0. The workspace (256-byte aligned) need not be cleared. wf_muon_plan: how such a call runs, plan[7]: matrices a
 * launch (what is left behind the last whole batch runs as a call of that many), 16-row tiles of the shorter side where everything runs on the
 * Gram matrix (1-4; then nothing follows), or 0; the tiling (0-2) and slices of the sum of X X^T, of its square, the update's tiling (0-3). */
int wf_muon_workspace(int64_t count, int64_t rows, int64_t cols, int64_t* bytes);
int wf_muon_plan(int64_t count, int64_t rows, int64_t cols, int* plan);
int wf_muon(const int64_t* table, int64_t count, int64_t rows, int64_t cols, int dt, double momentum, int nesterov, double keep,
            double rate, int steps, const double* coefficients, double eps, void* workspace, int64_t workspace_bytes, void* stream);
int wf_orthogonalize(const int64_t* table, int64_t count, int64_t rows, int64_t cols, int dt, int steps, const double* coefficients,
                     double eps, void* workspace, int64_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------------------- block streaming
 * Exact-size page-locked host memory: replaces PinnedHost's cudaHostRegister / cudaHostUnregister
 * (core/tiers/pinned.py:84-129); allocated page-locked (hipHostMalloc) instead of registered after the fact. */
int wf_host_alloc(size_t nbytes, void** ptr);
int wf_host_free(void* ptr);

/* Asynchronous host -> device copy on `stream`: replaces slot_flats[slot].copy_(host_flat, non_blocking=True)
 * (streaming/state.py:142-143). */
int wf_h2d_async(void* dst, const void* src, size_t nbytes, void* stream);

/* The side stream and the event fences of _StreamState (streaming/state.py:47-55,239-256;
 * streaming/activation.py:506-513). Streams are non-blocking at the default priority. wf_event_query returns 0
 * when the event's work is complete, 1 when not yet (the reference's event.query(), streaming/state.py:255). */
int wf_stream_create(void** stream);
int wf_stream_destroy(void* stream);
int wf_stream_synchronize(void* stream);
int wf_event_create(void** event, int timing);
int wf_event_destroy(void* event);
int wf_event_record(void* event, void* stream);
int wf_stream_wait_event(void* stream, void* event);
int wf_event_query(void* event);
int wf_event_synchronize(void* event);
int wf_event_elapsed_ms(void* start, void* end, float* ms);

/* ---------------------------------------------------------------------------------------------- GGUF files
 * The tensor table of a GGUF model file (version 2 or 3): the reference reads GGUF files through ComfyUI-GGUF /
 * gguf-py (not vendored; the files come from its tools/convert_to_gguf.py and llama.cpp's converters); these calls
 * give the SSD tier each tensor's absolute byte range so streamed blocks are read straight from the model file
 * (the role of file_block_layout / file_param_layout, core/tiers/plan.py:181-250, for GGUF instead of
 * safetensors). The file is untrusted: a malformed header is WF_EINVAL with a message, never a read out of
 * bounds. dims4: the tensor's dimensions, innermost first (GGUF order), padded with 1. Types: the GGML ids of
 * weightferry's formats plus F32 0, F16 1, BF16 30. */
int wf_gguf_open(const char* path, void** handle);
int wf_gguf_close(void* handle);
int wf_gguf_info(void* handle, int* version, int64_t* n_tensors, int64_t* n_kv, int64_t* alignment,
                 int64_t* data_offset, int64_t* file_bytes);
int wf_gguf_tensor(void* handle, int64_t i, char* name, int64_t name_cap, int* type, int* n_dims, int64_t* dims4,
                   int64_t* offset, int64_t* nbytes);
/* key/value i: type = GGUF value type (0-12); for arrays (9) elem_type and count; integers and bools in ival, floats
 * in fval (integers too), strings in sval (count = its length). */
int wf_gguf_kv(void* handle, int64_t i, char* key, int64_t key_cap, int* type, int* elem_type, int64_t* count,
               int64_t* ival, double* fval, char* sval, int64_t sval_cap);

/* ---------------------------------------------------------------------------------------------- SSD tier
 * A ring of `depth` host buffers filled by `threads` reader threads with streamed blocks read from the file at
 * `path`, in cyclic block order: the role of DiskRing (core/tiers/sources.py:165-355) with FileBlockSource /
 * PieceFileSource (:87-152), and, with wf_ring_submit / wf_ring_wait, of _SsdUploader (streaming/ssd_uploader.py:
 * 17-120). Block b is pieces piece_start[b] .. piece_start[b+1]-1: (file offset, bytes, offset in the packed block),
 * in increasing block offset. Flags: WF_RING_PINNED (page-locked buffers; required for submit), WF_RING_DIRECT
 * (O_DIRECT reads of 4 KiB aligned supersets through an aligned scratch buffer; ordinary reads where the file system
 * refuses). Consumers take blocks in the ring's order (block = position % n_blocks), either with acquire / release
 * from one thread (release's stream, if not NULL, must carry the copy out of the buffer: the buffer is refilled
 * after it), or with submit / wait: an uploader thread waits for the block, makes `stream` wait for `wait_event`,
 * copies into dst (dst_bytes >= the block), records `done_event` and returns the buffer to the readers; wait(ticket)
 * returns once that copy is on the stream (done_event recorded). A read or copy failure fails the ring: blocks read
 * before it are still served, later ones return an error until wf_ring_resync, which restarts the cycle at block 0
 * (no copies pending). */
#define WF_RING_PINNED 1
#define WF_RING_DIRECT 2
int wf_ring_open(const char* path, int64_t n_blocks, const int64_t* piece_start, const int64_t* piece_off,
                 const int64_t* piece_len, const int64_t* piece_dst, int depth, int threads, int flags, int device,
                 void** ring);
int wf_ring_acquire(void* ring, int64_t block, void** ptr, int64_t* nbytes, int* slot);
int wf_ring_release(void* ring, int slot, void* stream);
int wf_ring_submit(void* ring, int64_t block, void* dst, int64_t dst_bytes, void* wait_event, void* done_event,
                   void* stream, int64_t* ticket);
int wf_ring_wait(void* ring, int64_t ticket);
int wf_ring_resync(void* ring);
int wf_ring_stats(void* ring, double* read_s, double* wait_s, int64_t* bytes, int64_t* reads);
int wf_ring_close(void* ring);


#ifdef __cplusplus
}
#endif

#endif /* WEIGHTFERRY_H */
