// extern "C" surface of libmor_b200_mx (include/mor_b200_mx.h): argument validation, then one launch per operator.
#include "../../include/mor_b200_mx.h"

#include "mx_kernels.cuh"

using namespace morb;

namespace {

inline bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
// sizes the kernels index with 32-bit coordinates, and products of sizes that must not overflow 64 bits
inline bool too_large(int64_t v) { return v > 0x7FFFFF00; }

}  // namespace

extern "C" {

int mor_b200_mx_quantize_fp4(const void* input, int dtype, int64_t rows, int64_t cols, int64_t pitch, void* payload, void* scales,
                             void* stream) {
    if ((dtype != 0 && dtype != 1) || rows < 0 || cols <= 0 || pitch < cols) return kErrInvalidArgument;
    if (cols % 32) return kErrUnsupportedShape;
    if (rows == 0) return kOk;
    if (!input || !payload || !scales) return kErrInvalidArgument;
    if (too_large(rows) || too_large(cols) || pitch > (int64_t(1) << 31)) return kErrTooLarge;
    const int width = dtype == 1 ? 4 : 2;
    if (rows > 1 && (pitch * width) % 16) return kErrUnsupportedShape;
    if (!aligned(input, 16) || !aligned(payload, 4)) return kErrUnsupportedShape;
    return launch_quantize_fp4(input, dtype, rows, cols, rows == 1 ? cols : pitch, payload, static_cast<uint8_t*>(scales),
                               static_cast<cudaStream_t>(stream));
}

int mor_b200_mx_dequantize(const void* payload, const void* scales, void* out, int dtype, int64_t rows, int64_t cols, int block_cols,
                           int format, void* stream) {
    if ((dtype != 0 && dtype != 1) || rows < 0 || cols <= 0 || block_cols <= 0) return kErrInvalidArgument;
    if (format != kE4M3 && format != kE5M2 && format != kE2M3 && format != kE2M1) return kErrInvalidArgument;
    if (cols % block_cols) return kErrInvalidArgument;
    if (block_cols < 8 || block_cols > 256 || (block_cols & (block_cols - 1))) return kErrUnsupportedShape;
    if (rows == 0) return kOk;
    if (!payload || !scales || !out) return kErrInvalidArgument;
    if (too_large(rows) || too_large(cols)) return kErrTooLarge;
    if (!aligned(payload, 8) || !aligned(out, 16)) return kErrUnsupportedShape;
    return launch_dequantize(payload, static_cast<const uint8_t*>(scales), out, dtype, rows, cols, block_cols, format,
                             static_cast<cudaStream_t>(stream));
}

size_t mor_b200_mx_matmul_workspace_bytes(int64_t m, int64_t n, int64_t k, int a_format) {
    if (m <= 0 || n <= 0 || k <= 0 || k % 32 || too_large(m) || too_large(n) || too_large(k)) return 0;
    return mx_matmul_workspace(m, n, k, a_format == kE2M1);
}

int mor_b200_mx_matmul(const void* a, const void* a_scales, const void* b, const void* b_scales, int64_t m, int64_t n, int64_t k,
                       int a_format, int b_format, const void* bias, void* out, void* workspace, size_t workspace_bytes, void* stream) {
    if (m < 0 || n < 0 || k <= 0) return kErrInvalidArgument;
    const bool fp4 = a_format == kE2M1 && b_format == kE2M1;
    const bool fp8 = (a_format == kE4M3 || a_format == kE5M2) && (b_format == kE4M3 || b_format == kE5M2);
    if (!fp4 && !fp8) return kErrInvalidArgument;
    if (k % 32) return kErrUnsupportedShape;
    if (m == 0 || n == 0) return kOk;
    if (!a || !a_scales || !b || !b_scales || !out) return kErrInvalidArgument;
    if (too_large(m) || too_large(n) || too_large(k)) return kErrTooLarge;
    if (!aligned(a, 16) || !aligned(b, 16) || !aligned(a_scales, 16) || !aligned(b_scales, 16) || !aligned(out, 2) || !aligned(bias, 2))
        return kErrUnsupportedShape;
    const size_t need = mx_matmul_workspace(m, n, k, fp4);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return kErrWorkspace;
    const MxMatmulArgs x{a, b, static_cast<const uint8_t*>(a_scales), static_cast<const uint8_t*>(b_scales), bias, out, m, n, k, a_format, b_format, workspace};
    return launch_mx_matmul(x, static_cast<cudaStream_t>(stream));
}

int mor_b200_mx_matmul_grad(const void* g, int64_t g_pitch, const void* payload, const void* scales, int64_t m, int64_t n, int64_t k,
                            int format, int transpose_g, void* out, void* stream) {
    if (m < 0 || n < 0 || k < 0 || (transpose_g != 0 && transpose_g != 1)) return kErrInvalidArgument;
    if (format != kE4M3 && format != kE5M2 && format != kE2M3 && format != kE2M1) return kErrInvalidArgument;
    if (g_pitch < (transpose_g ? m : k)) return kErrInvalidArgument;
    if (n % 32) return kErrUnsupportedShape;
    if (too_large(m) || too_large(n)) return kErrTooLarge;
    if (m == 0 || n == 0) return kOk;
    if (k == 0) {   // an empty sum: the gradient of a batch without tokens
        if (!out) return kErrInvalidArgument;
        return cudaMemsetAsync(out, 0, (size_t)m * (size_t)n * 2, static_cast<cudaStream_t>(stream)) == cudaSuccess ? kOk : kErrLaunch;
    }
    if (!g || !payload || !scales || !out) return kErrInvalidArgument;
    if (too_large(k) || too_large(g_pitch)) return kErrTooLarge;
    if (g_pitch % 8 || !aligned(g, 16) || !aligned(payload, 16) || !aligned(out, 16)) return kErrUnsupportedShape;
    const MxGradArgs x{g, g_pitch, payload, static_cast<const uint8_t*>(scales), out, m, n, k, format, transpose_g};
    return launch_mx_grad(x, static_cast<cudaStream_t>(stream));
}

int mor_b200_mx_column_sums(const void* g, int64_t pitch, int64_t rows, int64_t cols, void* out, void* stream) {
    if (rows < 0 || cols < 0 || pitch < cols) return kErrInvalidArgument;
    if (cols == 0) return kOk;
    if (!out || (rows > 0 && !g)) return kErrInvalidArgument;
    if (too_large(rows) || too_large(cols) || too_large(pitch)) return kErrTooLarge;
    if ((rows > 1 && pitch % 8) || !aligned(g, 16) || !aligned(out, 2)) return kErrUnsupportedShape;
    return launch_column_sums(g, pitch, rows, cols, out, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
