/*
 * C ABI of the 8-bit linears of libSpMM_API.so for gfx950 (MI355X) and of the norm before them: products of 8-bit integers for
 * layers that are neither pruned (spmm_api.h) nor held in 4 bits (decode_api.h), in decode steps and, above all, over prompts.
 * None has a counterpart in the reference's library, whose dense linears are its FasterTransformer host's
 * (third_party/ft_spinfer.patch:3722-3753 is the call that the SpMM replaces there).
 *
 * Pointers, streams, graphs and return values as in decode_api.h: device memory, nothing allocated, no synchronisation, a
 * hipError_t as int, 1 with a message on stdout for arguments refused on the host.  An empty batch (N = 0) is a success that
 * launches nothing.  `dtype` is DECODE_FP16 or DECODE_BF16 of decode_api.h, the type of every 16-bit array of a call.
 *
 * 8-bit rows.  A row t of K numbers is held as codes int8 (-127..127) and one float32 scale:
 *   m = max |t_k|, code_k = the whole number nearest to 127 t_k / m (the even one of two), exactly; value_k = code_k * scale
 *   scale = m / 127, or m / 127 / rms where the norm below writes it
 * m below 2^-100: a row of zeros, codes and scale 0.  A row with an infinity or a NaN has codes 0 and scale NaN, and so NaN in
 * all that is computed from it.  Rows lie `stride` bytes apart, a multiple of 16, at most 2^28, 16-byte aligned, each readable up to K rounded
 * up to 16 bytes where a product reads them; what the bytes behind K hold does not matter.  What writes rows writes K bytes of each.
 */
#ifndef W8_API_H
#define W8_API_H

#include "decode_api.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Root-mean-square norm.  h = x + residual, rounded to `dtype` (residual NULL: h = x), t = h * weight,
 *   y = t / sqrt(mean(h^2) + eps)
 * rounded to `dtype` into y (codes NULL), or as 8-bit rows of t with scale m / 127 / sqrt(...) into codes and scales (y NULL).
 * h_out (NULL: not wanted) receives h; it and y may be x or the residual themselves (same address and stride), no output may overlap
 * an input or another output otherwise.  Rows of x, residual, h_out and y lie x_stride ... elements apart, at any alignment of the
 * type.  weight [K]; sums in float32; eps from 1e-20 up.  K from 1 to 2^24 (131071 for codes), N below 2^31. */
int RMS_Norm(hipStream_t stream, const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight,
             float eps, int N, int K, void* h_out, int64_t h_stride, void* y, int64_t y_stride, int8_t* codes,
             int64_t codes_stride, float* scales, int dtype);

/* 8-bit rows of x. */
int W8_Quantize(hipStream_t stream, const void* x, int64_t x_stride, int N, int K, int8_t* codes, int64_t codes_stride,
                float* scales, int dtype);

/* Weights, laid out once: codes int8 [M][K] (rows `stride` bytes apart, no alignment) and scales float32 [M] into `packed`,
 * W8_PackedBytes(M, K, 0) bytes, 16-byte aligned.  A second pair, up_codes not NULL, makes it the weights of a gated product:
 * W8_PackedBytes(M, K, 1) bytes.  M from 1 to 2^24, K from 1 to 131071 (a sum of K products stays in 32 bits).  0 bytes: sizes
 * that are refused. */
size_t W8_PackedBytes(int M, int K, int gated);
int    W8_Pack(hipStream_t stream, const int8_t* codes, int64_t stride, const float* scales, const int8_t* up_codes,
               int64_t up_stride, const float* up_scales, int M, int K, void* packed);

/* Y[n][m] = act(sum_k value(x)[n][k] * scale[m] code[m][k] + bias[m]), Y [N][M] contiguous in `dtype`, rounded once.  Sums of codes'
 * products are exact; they are turned into float32 and multiplied by the weight's scale, then by the row's.
 * W8_Gated: Y[n][m] = act(gate) * up, gate and up each such a sum over the two halves of gated weights, with gate_bias and up_bias.
 * x_scales NULL: x holds 16-bit rows (x_stride in elements, any alignment of the type) instead of 8-bit rows, which the call itself
 * turns into 8-bit rows in the workspace.  Biases NULL or [M] in `dtype`.  `activation`: 0 none, 1 ReLU, 2 GELU (tanh form), 3 SiLU
 * (x / (1 + exp(-x))).  N from 0 to 16 * 65535.  `workspace` must hold W8_WorkspaceBytes of the same sizes (NULL where that is 0),
 * 16-byte aligned, contents irrelevant; `x16` says that x holds 16-bit rows. */
#define W8_ACT_SILU 3
size_t W8_WorkspaceBytes(int M, int N, int K, int gated, int x16);
int    W8_Linear(hipStream_t stream, const void* packed, const void* x, int64_t x_stride, const float* x_scales, void* Y, int M,
                 int N, int K, const void* bias, int activation, void* workspace, size_t workspace_bytes, int dtype);
int    W8_Gated(hipStream_t stream, const void* packed, const void* x, int64_t x_stride, const float* x_scales, void* Y, int M,
                int N, int K, const void* gate_bias, const void* up_bias, int activation, void* workspace,
                size_t workspace_bytes, int dtype);

#ifdef __cplusplus
}
#endif

#endif /* W8_API_H */
