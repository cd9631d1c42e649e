/*
 * dsa_mi355x_layer.h -- C ABI of what stands between a model's residual stream
 * and its attention: root-mean-square norms (with the residual's addition, the
 * gradient, or an output of 8-bit codes) and products with 8-bit weights.  Part
 * of the same library as dsa_mi355x.h and of the same conventions: device
 * pointers, a stream, nothing allocated, no synchronisation, 0 / < 0 (invalid
 * argument, nothing enqueued) / > 0 (a hipError_t) with dsa_last_error().  No
 * reference counterpart: the reference takes q and kv as given (README.md:19-21).
 */
#ifndef DSA_MI355X_LAYER_H
#define DSA_MI355X_LAYER_H

#include <stdint.h>

#include "dsa_mi355x_cache.h" /* DSA_BF16, DSA_F16, DSA_F32 */

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Rows of x, with the residual added where it is given, normed:
 *   h = x + residual, rounded to their type;  inverse = 1 / sqrt(mean(h^2) + eps)
 *   y = h * inverse * weight
 * dsa_rms_norm writes y, rounded once to x's type.  dsa_rms_norm_fp8 writes the
 * 32-bit y as e4m3 codes with a scale for each block of 128 of a row (the last
 * block may be shorter):
 *   scale = max|y| / 448, pow2_scales: the least power of two not below that; 1 for
 *   a block of zeros;  code = e4m3(y / scale), to nearest even
 * and without weight the codes of h itself.  A block with a NaN has scale 1 (the NaN
 * its own code, the others e4m3(y), past 448 as 448); without one an infinity makes its
 * block's scale infinite, its own code NaN and the others 0.
 *
 *   x, residual [rows, dim], x_stride and residual_stride elements apart (at
 *   least 0, last stride 1); weight [dim] of x's type, or 32-bit (weight_f32)
 *   out [rows, dim] of x's type, or codes, of one byte each; sum [rows, dim]: h,
 *   unused without residual, where it must be given
 *   scales [rows, ceil(dim / 128)]; inverse [rows] 32-bit, or NULL
 * Outputs are contiguous and lie apart from the inputs.  dim at most
 * DSA_NORM_MAX_DIM; codes: a multiple of 16, out 16-byte aligned.  Sums are 32-bit; a
 * row whose squares leave their range, at either end, is multiplied by a power of two
 * first.  The inverse itself is held in 32 bits: infinite where it would pass 3.4e38,
 * of rows below 2.9e-39 with eps 0, whose gradients then are not finite.
 */
#define DSA_NORM_MAX_DIM 16384
typedef struct dsa_norm_args {
    const void* x;
    const void* residual;       /* or NULL */
    const void* weight;
    void* out;
    void* sum;
    float* scales;              /* dsa_rms_norm_fp8 */
    float* inverse;             /* dsa_rms_norm, or NULL */
    int64_t rows, x_stride, residual_stride;
    int32_t dim, dtype;         /* DSA_BF16, DSA_F16, DSA_F32 */
    int32_t weight_f32, pow2_scales;
    float eps;                  /* not negative */
    int32_t reserved;           /* zero */
} dsa_norm_args;
int dsa_rms_norm(const dsa_norm_args* args, void* stream);
int dsa_rms_norm_fp8(const dsa_norm_args* args, void* stream);

/*
 * Gradients of dsa_rms_norm, from h and the inverse that it wrote: with
 * u = h * inverse and b = grad_out * weight
 *   grad_in = (b - u * mean(b * u)) * inverse + grad_sum     (of x and the residual)
 *   grad_weight = sum over the rows of grad_out * u
 * h [rows, dim] h_stride apart; grad_out, grad_sum (or NULL), grad_in [rows, dim]
 * contiguous, of h's type; grad_weight [dim] of the weight's type, or NULL.  Outputs lie
 * apart from the inputs.
 * workspace: at least dsa_rms_norm_grad_ws_bytes(rows, dim) bytes, 16-byte aligned,
 * any contents; unused without grad_weight.  The order of the sums is fixed.
 */
typedef struct dsa_norm_grad_args {
    const void* h;
    const float* inverse;
    const void* weight;
    const void* grad_out;
    const void* grad_sum;
    void* grad_in;
    void* grad_weight;
    void* workspace;
    int64_t workspace_bytes, rows, h_stride;
    int32_t dim, dtype, weight_f32;
    int32_t reserved;           /* zero */
} dsa_norm_grad_args;
int64_t dsa_rms_norm_grad_ws_bytes(int64_t rows, int dim);
int dsa_rms_norm_grad(const dsa_norm_grad_args* args, void* stream);

/*
 * The product of 8-bit rows with 8-bit weights:
 *   out[m, n] = sum over blocks k of  a_scales[m, k] * b_scales[n / 128, k] *
 *               (sum over j in [128 k, min(128 k + 128, K)) of  a[m, j] * b[n, j])
 *
 *   a [M, K], b [N, K] e4m3 codes, 16-byte aligned, K a multiple of 16 below 2^20,
 *   M * N at most 2^37
 *   a_scales [M, ceil(K / 128)], b_scales [ceil(N / 128), ceil(K / 128)] 32-bit
 *   out [M, N] of type dtype, rounded once; sums are 32-bit, and so is the product of
 *   two scales, which has to be in their range.  For 16-bit outputs the
 *   matrix cores cut each product to 2^-13 of the largest of eight neighbours (an error
 *   of 1.5e-5 of a sum's size was measured), for DSA_F32 they are whole.
 */
typedef struct dsa_product_args {
    const uint8_t* a;
    const float* a_scales;
    const uint8_t* b;
    const float* b_scales;
    void* out;
    int32_t M, N, K;
    int32_t dtype;              /* DSA_BF16, DSA_F16, DSA_F32 */
} dsa_product_args;
int dsa_matmul_fp8(const dsa_product_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DSA_MI355X_LAYER_H */
