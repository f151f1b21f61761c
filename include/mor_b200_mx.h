/* C ABI of libmor_b200_mx: microscaled (MX) operands put to use on B200 (sm_100a).
 *
 * The operators of mor_b200.h quantise; these take the real quantised form further.  None has a counterpart in
 * boryiings/mor, whose operators only fake-quantize.  An MX matrix [rows, cols] is
 *   payload: one code per element -- a byte for E4M3 (format 0), E5M2 (1) and E2M3 (3; the code in the low six bits), as
 *            mor_b200_quantize_mx writes them (with MOR_B200_MX_OPERAND added to its format, for products), or half a byte for E2M1 (4): column 2j in bits 0-3, 2j + 1 in bits 4-7;
 *   scales:  one E8M0 byte for every `block_cols` consecutive columns of a row, row-major;
 *   element = decode(code) * 2^(scale - 127), NaN where the scale byte is 255.
 * All pointers are device pointers of the current device; tensors are row-major and, unless said otherwise, contiguous.
 * Calls enqueue on `stream`, do not synchronise, allocate or throw, and may be captured into a CUDA graph.  Status codes are those of mor_b200.h (0 ok, -1 invalid argument, -2 unsupported shape or alignment, -3
 * workspace missing or too small, -4 launch failed, -5 too large).  Sizes of zero in rows, m or n are valid and launch nothing.
 * A tile of a product whose operands did not arrive within the kernel's bounded wait is written as NaN. */
#ifndef MOR_B200_MX_H
#define MOR_B200_MX_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(_WIN32)
#define MOR_B200_MX_API
#else
#define MOR_B200_MX_API __attribute__((visibility("default")))
#endif

#define MOR_B200_MX_E2M1 4   /* beside MOR_B200_E4M3 (0), MOR_B200_E5M2 (1), MOR_B200_E2M3 (3) */

/* 4-bit quantisation, groups of 32.  input: bf16 (dtype 0) or float32 (dtype 1) [rows, cols] with `pitch` elements from
 * one row to the next, 16-byte aligned, pitch * element size a multiple of 16; cols a multiple of 32.  payload:
 * [rows, cols / 2], 4-byte aligned; scales: [rows, cols / 32].  The scale of a group is the largest power of two that
 * keeps its largest magnitude at or below 6 (the rule of mor_b200_quantize_mx, so nothing saturates); codes are rounded
 * to nearest even and keep the sign of zero.  A group of zeros gets byte 127, one that holds an infinity or a NaN gets
 * byte 255 and codes of zero. */
MOR_B200_MX_API int mor_b200_mx_quantize_fp4(const void* input, int dtype, int64_t rows, int64_t cols, int64_t pitch,
                                             void* payload, void* scales, void* stream);

/* Codes back to values: out is bf16 (dtype 0) or float32 (1) [rows, cols], 16-byte aligned; format 0, 1, 3 or 4.
 * block_cols: a power of two from 8 to 256 that divides cols; payload 8-byte aligned.  float32 values are exact (an
 * overflow is an infinity); bf16 values are rounded to nearest even, which only results below 2^-126 meet. */
MOR_B200_MX_API int mor_b200_mx_dequantize(const void* payload, const void* scales, void* out, int dtype, int64_t rows,
                                           int64_t cols, int block_cols, int format, void* stream);

/* out[m, n] = sum_k A[m, k] B[n, k] (+ bias[n]): both operands MX with groups of 32 along k, k a positive multiple of 32,
 * payloads and scales 16-byte aligned.  Formats: both E2M1, or each E4M3 or E5M2.  bias: bf16 [n] or NULL; out:
 * bf16 [m, n], 2-byte aligned.  Products and sums are formed by the tensor core in binary32, the bias is added in
 * binary32, and the result is rounded once.  m <= 64 takes a form in which tokens fill a narrow tile.  Sums that are
 * split over the CTAs of a cluster are added in a fixed order: results repeat bit for bit.
 * Large products need a workspace of mor_b200_mx_matmul_workspace_bytes(m, n, k, a_format) bytes (0 for the others, which
 * take NULL), 16-byte aligned, of any content.
 * Scale bytes lie in it in tensor-core order while the call runs, so calls that may overlap (other streams, captured
 * graphs) need one each. */
MOR_B200_MX_API size_t mor_b200_mx_matmul_workspace_bytes(int64_t m, int64_t n, int64_t k, int a_format);
MOR_B200_MX_API int mor_b200_mx_matmul(const void* a, const void* a_scales, const void* b, const void* b_scales, int64_t m,
                                       int64_t n, int64_t k, int a_format, int b_format, const void* bias, void* out,
                                       void* workspace, size_t workspace_bytes, void* stream);

/* out[m, n] = sum_k op(g)[m, k] W[k, n]: g is bf16 [m, k], or [k, m] with transpose_g, `g_pitch` elements from row to
 * row (g 16-byte aligned, g_pitch a multiple of 8); W is MX [k, n] with groups of 32 along n, n a multiple of 32, format
 * 0, 1, 3 or 4, payload 16-byte aligned; out: bf16 [m, n], 16-byte aligned.  With W the quantised weights [out, in] and g [tokens, out] this is
 * a linear layer's input gradient; with W the quantised input [tokens, in] and transpose_g its weight gradient.  W's
 * elements enter the product as bf16 (exact above 2^-126).  k = 0 gives zeros. */
MOR_B200_MX_API int mor_b200_mx_matmul_grad(const void* g, int64_t g_pitch, const void* payload, const void* scales, int64_t m,
                                            int64_t n, int64_t k, int format, int transpose_g, void* out, void* stream);

/* out[c] = sum_r g[r, c]: the gradient of a bias.  g: bf16 [rows, cols], `pitch` elements from row to row (16-byte aligned,
 * pitch a multiple of 8); out: bf16 [cols].  Sums in binary32 in a fixed order, rounded once; no rows give zeros. */
MOR_B200_MX_API int mor_b200_mx_column_sums(const void* g, int64_t pitch, int64_t rows, int64_t cols, void* out, void* stream);

#ifdef __cplusplus
}
#endif
#endif
