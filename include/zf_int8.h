/*
 * zf_int8.h -- C ABI of the 8-bit row operators: activations and weights held as int8 codes with one fp32 scale per row,
 * the add + RMS norm that writes them, the linear layer on them, and the two backward passes that read them instead of
 * the bf16 activations (8-bit activation checkpoints). The reference has no counterpart: its MLP is bf16 throughout and
 * its training forward keeps the activations in bf16 (ZipNeRFCudaBackend/ZipNeRFCudaBackend/mlp/src/nerf_mlp.cu:527-560).
 *
 * The format, int8 rows: codes int8 [n, d], scales float [n]; row r stands for the values codes[r, j] * scales[r].
 * Codes lie in [-127, 127]. Wherever codes are read or written their base is 16-byte aligned and their row stride is a
 * multiple of 16 bytes, at least d; the bytes between d and the stride are neither read as values nor written.
 *
 * Quantization of a row x with a = max |x_j|:
 *   scale = a / 127, or with power_of_two the smallest power of two that is no less; never below 2^-126;
 *   codes = x / scale, the fp32 quotient, rounded to nearest, ties to even (for scales of 2^102 and more a value within 2^-18
 *   of a half step may take either of its neighbours).
 *   a = 0: scale 0 and codes 0. A NaN or an infinity anywhere in the row: scale NaN and codes 0, so that every value read
 *   back from the row is NaN.
 * With a power-of-two scale every value codes * scale is a bf16 number (8 significant bits), so tensor-core operands
 * made from it carry no second rounding; the step is between 1 and 2 times a / 127.
 *
 * Conventions as zf_featurize.h: device pointers and sizes, work is only enqueued on the given stream, a failed call
 * returns its status and leaves the message in zf_last_error(). Strides are in elements; a pointer off its element's
 * alignment is refused. n = 0 is valid and launches nothing.
 */
#ifndef ZF_INT8_H
#define ZF_INT8_H

#include <stdint.h>

#include "zf_featurize.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { ZF_FLOAT32 = 0, ZF_BFLOAT16 = 1 };

/* codes and scales of the rows of x [n, d] (float or bf16, unit column stride, any row stride of at least d). */
typedef struct zf_quantize_rows_args {
    const void* x;
    int x_dtype;
    int64_t x_stride;
    int64_t n, d;
    int power_of_two;
    int8_t* codes;
    int64_t codes_stride;
    float* scales;
} zf_quantize_rows_args;
/* Quantizes rows; one launch. No counterpart in the reference. */
ZF_API int zf_quantize_rows(const zf_quantize_rows_args* args, struct CUstream_st* stream);

/* out [n, d] (float or bf16) = codes * scales, rounded once. */
typedef struct zf_dequantize_rows_args {
    const int8_t* codes;
    int64_t codes_stride;
    const float* scales;
    int64_t n, d;
    void* out;
    int out_dtype;
    int64_t out_stride;
} zf_dequantize_rows_args;
/* Restores rows; one launch. No counterpart in the reference. */
ZF_API int zf_dequantize_rows(const zf_dequantize_rows_args* args, struct CUstream_st* stream);

/* h = x + residual in fp32 (x alone without a residual), rstd = 1 / sqrt(mean_j(h^2) + eps), y = h * rstd * weight,
 * and y quantized by rows. sum receives h rounded to the residual's type (it may be the residual's own memory, with the
 * same stride); x must not overlap any output. weight (float [d]) may be NULL: the codes then hold the normalised rows
 * themselves, which is what zf_rms_norm_int8_backward reads (a gain goes into the columns of the next layer's weight).
 * eps > 0. Rows whose squares sum past fp32's range are treated like rows with an infinity. */
typedef struct zf_rms_norm_int8_args {
    const void* x;
    int x_dtype;
    int64_t x_stride;
    const void* residual;      /* [n, d], or NULL */
    int residual_dtype;
    int64_t residual_stride;
    const float* weight;       /* [d], or NULL */
    int64_t n, d;
    float eps;
    int power_of_two;
    int8_t* codes;
    int64_t codes_stride;
    float* scales;
    void* sum;                 /* [n, d] in the residual's type; NULL exactly when residual is */
    int64_t sum_stride;
    float* rstd;               /* [n], or NULL */
} zf_rms_norm_int8_args;
/* The add + RMS norm with 8-bit output; one launch. No counterpart in the reference. */
ZF_API int zf_rms_norm_int8(const zf_rms_norm_int8_args* args, struct CUstream_st* stream);

/* The norm's backward from its own 8-bit output: with y = codes * scales (the forward without a weight),
 *   grad_x = rstd * (grad - y * mean_j(grad * y)) + grad_residual,
 * the gradient of both x and the residual (straight through the quantization). grad [n, d] is the gradient of y;
 * grad_residual (the residual stream's own gradient) may be NULL. grad_x has grad_residual's type, else grad's, and may
 * be the memory of either when type and stride agree. */
typedef struct zf_rms_norm_int8_backward_args {
    const void* grad;
    int grad_dtype;
    int64_t grad_stride;
    const int8_t* codes;
    int64_t codes_stride;
    const float* scales;
    const float* rstd;
    const void* grad_residual; /* [n, d], or NULL */
    int grad_residual_dtype;
    int64_t grad_residual_stride;
    int64_t n, d;
    void* grad_x;
    int64_t grad_x_stride;
} zf_rms_norm_int8_backward_args;
/* The norm's backward from its codes; one launch. No counterpart in the reference. */
ZF_API int zf_rms_norm_int8_backward(const zf_rms_norm_int8_backward_args* args, struct CUstream_st* stream);

/* output [n, out] = scales[r] * weight_scales[o] * (codes [n, in] @ weight_codes [out, in]^T) + bias[o], the products
 * summed exactly in 32-bit integers, then optionally ReLU (a NaN stays a NaN), rounded once to float or bf16.
 * in <= 131071 (so that no sum leaves 32 bits, codes of -128 included); n and out below 2^31 - 256. status: a device int
 * that the kernel sets to 1 if one of its bounded waits ran out, which leaves this launch's output undefined. */
typedef struct zf_int8_linear_args {
    const int8_t* codes;
    int64_t codes_stride;
    const float* scales;
    const int8_t* weight_codes;
    int64_t weight_stride;
    const float* weight_scales;
    const float* bias;         /* [out], or NULL */
    int64_t n, in, out;
    int relu;
    void* output;
    int output_dtype;
    int64_t output_stride;
    int* status;
} zf_int8_linear_args;
/* The 8-bit linear layer; one launch. The bf16 counterpart is a cuBLASLt layer of NerfMlp::forward (nerf_mlp.cu:503-560). */
ZF_API int zf_int8_linear(const zf_int8_linear_args* args, struct CUstream_st* stream);

/* The weight gradient of a linear layer from the 8-bit checkpoint of its input:
 *   grad_weight [out, in] (contiguous float) += sum_r grad[r, o] * (codes[r, k] * scales[r]),
 *   grad_bias [out] (float, or NULL) += sum_r grad[r, o].
 * grad [n, out] bf16, any row stride of at least out. codes * scales is rounded to bf16 for the tensor cores: exact for
 * power-of-two scales, one rounding for others. The sums run in a fixed order: the same call gives the same bits.
 * workspace: zf_int8_weight_grad_workspace_size(n, in, out) bytes, 16-byte aligned. status: as zf_int8_linear. */
typedef struct zf_int8_weight_grad_args {
    const uint16_t* grad;
    int64_t grad_stride;
    const int8_t* codes;
    int64_t codes_stride;
    const float* scales;
    int64_t n, in, out;
    float* grad_weight;
    float* grad_bias;          /* [out], or NULL */
    void* workspace;
    int64_t workspace_bytes;
    int* status;
} zf_int8_weight_grad_args;
/* Bytes of the workspace. No counterpart in the reference. */
ZF_API int64_t zf_int8_weight_grad_workspace_size(int64_t n, int64_t in, int64_t out);
/* The weight gradient from 8-bit codes. The bf16 counterpart is a weight-gradient GEMM of NerfMlp::backward
 * (nerf_mlp.cu:583-607). */
ZF_API int zf_int8_weight_grad(const zf_int8_weight_grad_args* args, struct CUstream_st* stream);

#ifdef __cplusplus
}
#endif

#endif
