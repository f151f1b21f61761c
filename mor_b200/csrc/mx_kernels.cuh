// Launch functions of libmor_b200_mx, one per operator.  Each returns a status code (common.cuh) and never synchronises,
// allocates or throws.  Arguments have been checked by the caller (mx_api.cu).
#pragma once

#include "kernels.cuh"

namespace morb {

enum : int { kE2M1 = 4 };   // beside Fmt: two codes to a byte

// mx_quant.cu
int launch_quantize_fp4(const void* in, int is_fp32, int64_t rows, int64_t cols, int64_t pitch, void* payload, uint8_t* scales, cudaStream_t st);
int launch_dequantize(const void* payload, const uint8_t* scales, void* out, int out_fp32, int64_t rows, int64_t cols, int bcols, int fmt, cudaStream_t st);
// out[c] = sum_r g[r, c], bf16, rows `pitch` elements apart
int launch_column_sums(const void* g, int64_t pitch, int64_t rows, int64_t cols, void* out, cudaStream_t st);

// mx_matmul.cu: out[m, n] = sum_k a[m, k] b[n, k] + bias[n]
struct MxMatmulArgs {
    const void *a, *b;
    const uint8_t *a_scales, *b_scales;
    const void* bias;   // bf16 [n] or null
    void* out;          // bf16 [m, n]
    int64_t m, n, k;
    int a_fmt, b_fmt;
    void* workspace;    // mx_matmul_workspace bytes
};
size_t mx_matmul_workspace(int64_t m, int64_t n, int64_t k, int fp4);
int launch_mx_matmul(const MxMatmulArgs& a, cudaStream_t st);

// mx_grad.cu: out[m, n] = sum_k op(g)[m, k] decode(payload)[k, n]
struct MxGradArgs {
    const void* g;      // bf16 [m, k], or [k, m] where across
    int64_t g_pitch;    // elements
    const void* payload;
    const uint8_t* scales;
    void* out;          // bf16 [m, n]
    int64_t m, n, k;
    int fmt, across;
};
int launch_mx_grad(const MxGradArgs& a, cudaStream_t st);

}  // namespace morb
