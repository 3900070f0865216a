/*
 * mi355_train.h - C ABI of the training operators in libmi355_aten.so: layer norm's backward pass, the gated
 * linear projection of a feed-forward block with its backward pass, and dropout from a counter-based generator
 * with the residual add.  Conventions, status codes and dtypes are those of mi355_aten.h: device pointers, extents
 * and strides in elements, kernels only enqueued on `stream`, nothing launched on error, 0 on success.
 */
#ifndef MI355_TRAIN_H
#define MI355_TRAIN_H

#include "mi355_aten.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- layer norm, backward ---------------------------------------------------------- */

/* For M dense rows of N elements, with xhat = (x - mean) * rstd and g = dy * weight (weight NULL: g = dy):
 *   dx = rstd * (g - mean_N(g) - xhat * mean_N(g * xhat)),  dweight = sum_M dy * xhat,  dbias = sum_M dy.
 * Any of dx, dweight, dbias may be NULL (not wanted).  dy, x, dx: `dtype` (f32, f16, bf16, f64); weight, dweight,
 * dbias: `w_dtype` (dtype, or f32 for f16 / bf16 rows); mean, rstd: M values each, f32 (f64 for f64 rows).  Sums are
 * held in fp32 (fp64 for f64 rows) and added in a fixed order: the same call gives the same bits.
 * The workspace (contents undefined before and after) must hold mi355_layer_norm_backward_workspace_bytes() bytes,
 * 16-byte aligned (0 for a handful of rows: NULL is accepted); a call with less is refused.
 * Slot: native_layer_norm_backward__default. */
int64_t mi355_layer_norm_backward_workspace_bytes(int64_t M, int64_t N, int dtype);
int mi355_layer_norm_backward(const void* dy, const void* x, int dtype, const void* mean, const void* rstd,
                              const void* weight, int w_dtype, void* dx, void* dweight, void* dbias, int64_t M, int64_t N,
                              void* workspace, int64_t workspace_bytes, void* stream);

/* ---- gated linear projection ------------------------------------------------------- */

typedef enum mi355_activation {
  MI355_SILU = 0,      /* g / (1 + exp(-g))                                         */
  MI355_GELU = 1,      /* g * Phi(g), Phi the normal distribution function          */
  MI355_GELU_TANH = 2  /* g / 2 * (1 + tanh(sqrt(2 / pi) * (g + 0.044715 g^3)))     */
} mi355_activation;

/* h = act(x Wg^T) * (x Wu^T) in one kernel: x [M][K] with rows x_rs apart (one row: any x_rs), weight [2F][K] = [Wg; Wu] with
 * rows w_rs apart, both unit-stride along K; h [M][F] dense; pre (may be NULL) receives the pre-activations [M][2F], dense.  All of
 * `dtype` (f32, f16, bf16, f64).  Products accumulate in fp32 (fp64 for f64); the activation takes the unrounded sums.
 * Any strides and alignment: with K >= 8 up to 64 rows of f16 or bf16, 32 of f32; with any K 2 of f16 or bf16, 4 of f32, 8
 * of f64.  More rows of f16 and bf16 with 16-byte aligned rows and K % 128 == 0, or K % 64 == 0 and at most 512 tiles of
 * 128 rows by 64 features.  Otherwise MI355_ERR_UNSUPPORTED with nothing launched: mi355_pad_rows brings f16 and bf16 operands into rows that are
 * taken; more rows of f32 and f64 are a product followed by mi355_gated_act. */
int mi355_gated_linear(const void* x, int64_t x_rs, const void* weight, int64_t w_rs, void* h, void* pre, int64_t M, int64_t F,
                       int64_t K, int act, int dtype, void* stream);

/* dst [R][ld] = src [R][C] with rows src_rs apart at any alignment, columns C .. ld - 1 zeros, elements of 2 or 4 bytes moved
 * as bits; dst and its rows start on 16-byte boundaries.  It brings x and weight into rows that the kernels take. */
int mi355_pad_rows(const void* src, int64_t src_rs, int64_t R, int64_t C, void* dst, int64_t ld, int element_size, void* stream);

/* h[m][f] = act(pre[m][f]) * pre[m][F + f] from dense pre [M][2F], f32 or f64: the activation behind a product. */
int mi355_gated_act(const void* pre, void* h, int dtype, int64_t M, int64_t F, int act, void* stream);

/* The gated projection's gradients: dpre = [dh * up * act'(gate) | dh * act(gate)] with gate = pre[m][f], up = pre[m][F + f], rounded once to
 * `dtype` (f32, f16, bf16, f64), then dx [M][K] = dpre W and dweight [2F][K] = dpre^T x, accumulated in fp32 (fp64).
 * (f16: dpre beyond 65504 becomes infinite, and with it its row of dx and of dweight.)  dh [M][F], pre [M][2F], dx and
 * dweight are dense; x and weight have rows x_rs and w_rs apart (one row of x: any x_rs).  dx or dweight may be NULL.
 * The workspace (16-byte aligned, contents undefined before and after; not shared by calls that may overlap in time)
 * holds dpre and the products' scratch, or partial sums of dx: mi355_gated_linear_backward_workspace_bytes() always suffices. */
int64_t mi355_gated_linear_backward_workspace_bytes(int64_t M, int64_t F, int64_t K, int dtype);
int mi355_gated_linear_backward(const void* dh, const void* x, int64_t x_rs, const void* weight, int64_t w_rs, const void* pre,
                                void* dx, void* dweight, int64_t M, int64_t F, int64_t K, int act, int dtype,
                                void* workspace, int64_t workspace_bytes, void* stream);

/* ---- dropout with a residual ------------------------------------------------------- */

/* out[i] = residual[i] + (draw_i >= t ? x[i] * 65536 / (65536 - t) : 0), t = round(p * 65536) with halves to the even
 * neighbour, over n dense elements (residual NULL: 0).  draw_i is 16 bits of Philox-4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as
 * easy as 1, 2, 3", 2011): key = the 64-bit seed, counter = offset + i / 8, bits 16 (i % 8) .. + 15 of its 128 output
 * bits.  `rng` (device memory, two int64: seed, offset) is read by the kernel when it is not NULL, so that a captured
 * graph draws anew after the caller has advanced it; otherwise seed and offset are used.  n elements use up
 * (n + 7) / 8 counters.  The same draws with x = dy and no residual give the gradient.  A dropped x is not read into
 * the result, whatever it holds. */
int mi355_dropout_add(const void* x, const void* residual, int dtype, double p, const void* rng, int64_t seed, int64_t offset,
                      void* out, int64_t n, void* stream);

#ifdef __cplusplus
}
#endif
#endif
