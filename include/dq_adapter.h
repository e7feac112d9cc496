/* dq_adapter.h -- low-rank adapters of many requests beside the quantized
 * linears (same library as dq_linear.h), forward and backward, and the 8-bit
 * activation checkpoints that the backward pass reads.
 *
 * Layouts (bf16 unless said otherwise, row-major, device pointers):
 *   x      [M, K]      activations, row stride ldx
 *   y      [M, N]      the shared projection's output, row stride ldy
 *   down   [A, r, K]   every adapter's down projection (its first factor)
 *   up     [A, r, N]   every adapter's up projection, laid out with its N
 *                      output features contiguous (the transpose of the
 *                      [N, r] factor that checkpoints store), so that the
 *                      backward pass reads both factors as the forward does
 *   scale  f32 [A]     per-adapter factor (alpha / r)
 * K, N and r are multiples of 8, r <= 128; row strides are multiples of 8 and
 * every operand 16-byte aligned.  The reference has no adapters. */
#ifndef DQ_ADAPTER_H
#define DQ_ADAPTER_H

#include "dq_linear.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The tokens of a batch sorted by adapter, built on the device once per batch
 * and read by every dq_adapter_* call on it (each layer, forward and
 * backward).  Request i holds tokens offsets[i] .. offsets[i + 1] - 1 (int32
 * [R + 1], not decreasing, within 0..M) and uses adapter ids[i] (int32 [R];
 * -1: none; the same adapter any number of times).  Tokens outside every
 * request have no adapter.  Both arrays are device memory and are not read by
 * the host.  An id outside -1..A-1 counts as none, and offsets that decrease
 * or leave 0..M leave every token without an adapter; either is recorded as
 * DQ_ERR_INDEX for dq_device_error.  M <= 2^30, 1 <= A <= 65535, 0 <= R <= 2^20.
 * The plan buffer (dq_adapter_plan_bytes) is 16-byte aligned and needs no
 * initialization; it may be rebuilt in place, also inside a captured graph,
 * as long as M, R and A stay the same. */
size_t dq_adapter_plan_bytes(int64_t M, int64_t R, int A);
int dq_adapter_plan(const int32_t* ids, const int32_t* offsets, int64_t R, int64_t M, int A,
                    void* plan, size_t plan_bytes, dq_stream_t stream);

/* out[m] = act(y[m] + scale_a * (x[m] . down_a^T) . up_a) for each token m of
 * the plan's M with its adapter a; act(y[m]) where it has none.  out may be y
 * (then tokens without an adapter are left as they are unless act or hidden
 * asks for them).  act as dq_linear_*_ex; with a gated activation up's and y's
 * columns are in the gated row order, N % 32 == 0 and out has N / 2 columns.
 * hidden (or NULL): bf16 [M, r], receives scale_a * x . down_a^T (zero rows
 * where there is none), which the backward pass takes.  Apart from y, out
 * overlaps no operand (dx_out below: apart from dx).
 * The sums of the down projection are kept in float32 over K, rounded once
 * to bf16 for the up projection, which accumulates in float32 onto y; out is
 * rounded once.  The workspace (16-byte aligned, at most M * r * 2 bytes; none
 * for small batches) is needed only where hidden is NULL. */
size_t dq_adapter_add_workspace(int64_t M, int64_t R, int r, int A);
int dq_adapter_add(const void* y, int64_t ldy, const void* x, int64_t ldx, int64_t M, int64_t R,
                   int64_t K, int64_t N, const void* down, const void* up, const float* scale, int r,
                   int A, const void* plan, int act, void* out, int64_t ldo, void* hidden,
                   void* workspace, size_t workspace_bytes, dq_stream_t stream);

/* The gradients of dq_adapter_add without an activation.  With
 * g[m] = scale_a * dy[m] . up_a^T:
 *   dx_out[m] = dx[m] + g[m] . down_a           (dx_out may be dx)
 *   ddown[a]  = sum over a's tokens of g^T x    [A, r, K]
 *   dup[a]    = sum over a's tokens of hidden^T dy   [A, r, N]
 * hidden as dq_adapter_add wrote it.  x is bf16 [M, K] (x_scales NULL), or the
 * int8 codes [M, K] of a checkpoint with its scales f32 [M, ceil(K / 128)]
 * (row stride ceil(K / 128)); K % 16 == 0 then.  Adapters without tokens get
 * zero gradients.  ddown and dup may be NULL together (input gradient only; x
 * and hidden are not read then), or dx and dx_out (the factors' gradients only,
 * as for a first layer; the product with down is left out then).  Sums are float32 in a fixed order: the same
 * inputs give the same bits. */
size_t dq_adapter_backward_workspace(int64_t M, int64_t R, int64_t K, int64_t N, int r, int A);
int dq_adapter_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx,
                        const float* x_scales, const void* hidden, int64_t M, int64_t R, int64_t K,
                        int64_t N, const void* down, const void* up, const float* scale, int r, int A,
                        const void* plan, const void* dx, int64_t lddx, void* dx_out, int64_t lddxo,
                        void* ddown, void* dup, void* workspace, size_t workspace_bytes,
                        dq_stream_t stream);

/* An activation kept in 8 bits until the backward pass.  Per row and run of
 * 128 features (the last may be shorter): scale = max(max|x|, 1e-12) / 127
 * (f32), codes = rint(x / scale) (ties to even), int8.  A run that holds a NaN
 * or an infinity gets a NaN scale, so all of it is restored as NaN.
 * x bf16 [M, K] (row stride ldx), codes [M, K], scales [M, ceil(K / 128)];
 * K % 16 == 0, ldx % 8 == 0. */
int dq_checkpoint_pack(const void* x, int64_t ldx, int64_t M, int64_t K, int8_t* codes,
                       float* scales, dq_stream_t stream);
/* out[m, k] = bf16(codes * scale), row stride ldo. */
int dq_checkpoint_unpack(const int8_t* codes, const float* scales, int64_t M, int64_t K, void* out,
                         int64_t ldo, dq_stream_t stream);

/* Input gradient of the quantized linears: dx[M, K] = dy[M, N] . dequant(W),
 * W as dq_linear_nf4 / dq_linear_fp8 take it (absmax f32 or, scale_dtype
 * DQ_DTYPE_BF16, bf16).  Up to 256 tokens, and up to 512 where N >= 2048, the
 * weight is decoded next to the product, in one launch without a workspace;
 * beyond, once, transposed, into the workspace (16-byte aligned) and
 * multiplied by the bf16 CTA-pair GEMM.  dq_linear_dgrad_workspace_for: the
 * bytes that a call with M tokens needs (0: none, workspace may be NULL);
 * dq_linear_dgrad_workspace: enough for any number of tokens.  Sums are float32, dx is
 * rounded once; the same inputs give the same bits.  N % 8 == 0, K % 64 == 0
 * (NF4) or K % 16 == 0 (fp8); dy and dx contiguous, 16-byte aligned. */
size_t dq_linear_dgrad_workspace_for(int64_t M, int64_t N, int64_t K);
size_t dq_linear_dgrad_workspace(int64_t N, int64_t K);
int dq_linear_nf4_dgrad(const void* dy, int64_t M, int64_t N, const uint8_t* packed,
                        const void* absmax, int scale_dtype, int64_t K, void* dx, void* workspace,
                        size_t workspace_bytes, dq_stream_t stream);
int dq_linear_fp8_dgrad(const void* dy, int64_t M, int64_t N, const uint8_t* w8, float scale,
                        int64_t K, void* dx, void* workspace, size_t workspace_bytes,
                        dq_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* DQ_ADAPTER_H */
