/*
 * mesh_moe_fp8.h -- C ABI of the part of libmesh_moe_hip.so that works on 8-bit
 * operands: products of e4m3 numbers with a scale for each block of 128, the passes
 * that make such operands, and the RMS norm that writes its result as one.
 *
 * The conventions are those of mesh_moe.h: device pointers owned by the caller, one
 * asynchronous call on `stream`, 0 or a negative MESH_MOE_E_* code, the reason from
 * mesh_moe_last_error().  Nothing is allocated or kept between calls: every call can
 * be recorded into a HIP graph, and calls on different streams do not meet unless they
 * share a workspace or an output.
 *
 * An 8-bit operand with `rows` rows of K values (K being the reduction index of the
 * product it is made for) is
 *   values [rows, KP]  e4m3 (one sign, four exponent, three mantissa bits; no
 *                      infinity), KP = K rounded up to whole blocks of 128; the
 *                      values from K on are zeros
 *   scales [rows, KS]  one byte per block, KS = KP / 128 rounded up to a multiple of
 *                      4 (bytes of blocks that a row does not have may hold anything)
 * and value i of a row stands for values[i] * 2^(scales[i / 128] - 127).  A block's
 * exponent is the smallest, from -117 on, for which its largest magnitude is at most
 * 448 (the largest e4m3 number) times 2^exponent; values are rounded to the nearest,
 * ties to even.  Powers of two leave the mantissas as they are, they are what the
 * matrix instructions of gfx950 take, and what 8-bit values stand for is a number of
 * bfloat16 too.  Below -117 it would not be; values under 2^-127 become zeros or
 * multiples of 2^-126 instead.  A block with an infinity or a NaN is NaN as a whole
 * (scale byte 127).
 * Products take scale bytes from 10 (which is -117) on, 255 making a block NaN; blocks
 * with a byte below, which no call here makes, they may count as zeros.
 * What a launch of 2^32 threads cannot cover (8 million tiles of few rows, 16 million
 * tiles of 128 x 128 to quantize) is refused, MESH_MOE_E_UNSUPPORTED.
 *
 * The reference has no 8-bit arithmetic; the calls are forms of what it does in
 * float32 or bfloat16, which is named at each.
 */
#ifndef MESH_MOE_FP8_H_
#define MESH_MOE_FP8_H_

#include "mesh_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* (counted up with every change of a declaration, and of what a call accepts) */
#define MESH_MOE_FP8_ABI_VERSION 3

int mesh_moe_fp8_abi_version(void);

/*
 * A tensor's rows, its columns or both as 8-bit operands, in one pass over it.
 *   x [E,R,K] dtype
 *   relu_mask [E,R,K] dtype or NULL: elements whose mask is not positive count as 0
 *     (the gradient behind a ReLU whose output is the mask, mesh_tensorflow/ops.py:
 *     1818-1921)
 *   row_count [E] int32 or NULL: rows from row_count[e] on (clamped to 0 .. R) count
 *     as zeros
 *   row_values [E,R,KP], row_scales [E,R,KS]: for products over K; or both NULL
 *   column_values [E,K,RP], column_scales [E,K,RS] (RP, RS from R as KP, KS from K):
 *     the transposed tensor, for products over R; or both NULL.  Of a weight [E,K,N]
 *     these are what mesh_moe_fp8_expert_linear multiplies by, as
 *     mesh_moe_pack_weights lays out a bf16 one (the rows: what the gradient of its
 *     input needs).
 */
int mesh_moe_fp8_quantize(const void* x, const void* relu_mask,
                          const int32_t* row_count, void* row_values,
                          uint8_t* row_scales, void* column_values,
                          uint8_t* column_scales, int E, int R, int K, int dtype,
                          void* stream);

/*
 * What an operand stands for: y[r, i] = values[r, i] * 2^(scales[r, i / 128] - 127),
 * i < K; NaN where the scale byte is 255.  Exact in float32, and from scale byte 3 on in
 * bfloat16, below it rounded to it (but for numbers from 2^128 on, which float32 values
 * from 248 * 2^120 on round to: infinities here).
 *   values [rows,KP], scales [rows,KS]; y [rows,K] dtype
 */
int mesh_moe_fp8_dequantize(const void* values, const uint8_t* scales, void* y,
                            int64_t rows, int K, int dtype, void* stream);

/*
 * RMS norm with the residual's addition, its result as an 8-bit operand
 * (sublayer_residual, sublayer_rms_norm and sublayer_mask_padding,
 * mesh_tensorflow/transformer/transformer.py:584-587, :493-516, :469-489):
 *   sum = x + residual (rounded to dtype: it is the next residual)
 *   y = sum * rsqrt(mean(sum^2) + epsilon) * scale * row_mask[row], in float32 (0 in
 *     rows whose mask is 0, whatever they hold)
 * and y is rounded once, to e4m3 (mesh_moe_residual_rms_norm rounds every step to
 * dtype, as the reference's operations do).
 *   x, residual, sum [rows,M] dtype (residual and sum may be NULL together: the norm
 *   of x); scale [M] dtype; row_mask [rows] dtype or NULL
 *   values [rows,MP], scales [rows,MS]; norm [rows,M] dtype or NULL: y rounded to dtype
 *   (what a training step makes the columns from)
 */
int mesh_moe_fp8_residual_rms_norm(const void* x, const void* residual,
                                   const void* scale, const void* row_mask, void* sum,
                                   void* norm, void* values, uint8_t* scales,
                                   int64_t rows, int M, double epsilon, int dtype,
                                   void* stream);

/*
 * One projection per expert (a dense layer with E = 1) of 8-bit operands:
 *   y[e] = act(a[e] . w[e]^T), float32 sums on the matrix instructions
 * (mtf.layers.dense with expert_dims, mesh_tensorflow/layers.py:129-208, as
 * mesh_moe_expert_linear does it in bf16).
 *   a_values [E,R,KP], a_scales [E,R,KS]; w_values [E,N,KP], w_scales [E,N,KS]
 *   row_count [E] int32 or NULL: only the first row_count[e] rows of expert e (clamped
 *     to 0 .. R) are multiplied; the others of y are left as they are
 *   y_scales NULL: y [E,R,N] bf16.  Otherwise y [E,R,NP] and y_scales [E,R,NS] are an
 *     8-bit operand for a product over N, rounded once from the float32 result
 *   workspace: mesh_moe_fp8_expert_linear_workspace_bytes bytes, which may be 0
 * Values, y where it is an 8-bit operand, and the workspace lie on 16 bytes, scales on 4.
 *
 * Precision: the matrix instructions for 8 bits cut the products of 8 neighbouring values
 * off, towards zero, below 2^-13 of the power of two in the largest of them (e4m3 numbers
 * below the normal ones count as 2^-6 there), and add up in float32.  A sum loses less than
 * 2^-10 of its products' magnitudes, with normally distributed operands about 2^-14 of
 * itself; an 8-bit result may lie a whole step from the exact one's.  Where products of at
 * most 128 rows are bound by other things they are multiplied in bf16, which is exact, and
 * float32 additions are all that is lost.  mesh_moe_fp8_expert_linear_exact tells (1 or 0;
 * eight_bit: the kind of result, counted: row_count is given) which sizes that is so for.
 * It goes by what is estimated to be faster: one row's bits may depend on the number of
 * rows, experts and columns beside it.
 */
int mesh_moe_fp8_expert_linear_exact(int E, int R, int K, int N, int eight_bit,
                                     int counted);
size_t mesh_moe_fp8_expert_linear_workspace_bytes(int E, int R, int K, int N,
                                                  int eight_bit);
int mesh_moe_fp8_expert_linear(const void* a_values, const uint8_t* a_scales,
                               const void* w_values, const uint8_t* w_scales,
                               const int32_t* row_count, void* y, uint8_t* y_scales,
                               int E, int R, int K, int N, int activation,
                               void* workspace, size_t workspace_bytes, void* stream);

/*
 * The gradients of such a projection (EinsumOperation.gradient,
 * mesh_tensorflow/ops.py:2846-2854), with the gradient of its output made an 8-bit
 * operand along either index first (dz = dy, or dy where relu_mask is positive):
 *   da[e] = dz[e] . w[e],  dw[e] = a[e]^T . dz[e]
 *   a_column_values [E,K,RP], a_column_scales [E,K,RS]: the columns of a, finite in rows
 *     from row_count on
 *   dy [E,R,N] dtype; relu_mask [E,R,N] dtype or NULL; row_count as above: rows of dy
 *   behind it count as zeros, and those of da are left as they are
 *   w_row_values [E,K,NP], w_row_scales [E,K,NS]: the rows of w [E,K,N]; NULL
 *   together with da where da is not wanted
 *   da [E,R,K] bf16, dw [E,K,N] bf16
 * Same alignment as above.
 */
size_t mesh_moe_fp8_expert_linear_backward_workspace_bytes(int E, int R, int K, int N,
                                                           int want_da);
int mesh_moe_fp8_expert_linear_backward(
    const void* a_column_values, const uint8_t* a_column_scales, const void* dy,
    const void* relu_mask, const int32_t* row_count, const void* w_row_values,
    const uint8_t* w_row_scales, void* da, void* dw, int E, int R, int K, int N,
    int dtype, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif  /* MESH_MOE_FP8_H_ */
